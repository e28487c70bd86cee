// Attention over the paged cache held in 4 bits (its layout: cache_ops.h).  Of a row (a token and a head) at position i of a request:
//   s_j = scale * q . k_j over the tokens j it sees (i - window < j <= i, in a page that the table has),  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).
// With k_j = a_j c_j + b_j and v_j = a'_j c'_j + b'_j (codes c of 0 .. 15, a step a and a lowest value b of the token's head):
//   s_j = scale * (a_j (q . c_j) + b_j sum(q)),   out = (sum_j (p_j a'_j) c'_j + sum_j p_j b'_j) / sum_j p_j,
// so the matrix instructions multiply codes.  A code in bits 0 .. 3 or 4 .. 7 of a half is the fp16 c 2^-24 or c 2^-20 (a number below the normal
// ones, which they take as it is): eight codes of a 32-bit word become four pairs with four ands and one shift, and what is multiplied with the second kind is
// 2^-4 of itself.  q goes in as fp16 times a power of two per row that takes its largest element below 2^14: exactly, but for what is 2^-28 of it.
// p_j a'_j is rounded to fp16 (2^-11 of it), with a power of two per wavefront that keeps the largest a' so far below 2^14; p of odd tokens times 2^-4.  All sums and the
// statistics are in 32 bits.
//
// A wavefront takes blocks of 64 tokens.  Keys: lane (m, g) = (lane % 16, lane / 16) loads a quarter g of token m of each of four tiles, which is the
// left operand of  scores[token][row];  so a lane gets the scores of tokens 4 g .. 4 g + 3 of each tile for row m, and what it makes of them is the right
// operand of  out[element][row]  as it stands.  Its left operand, 16 tokens of one element per lane, is read out of LDS by ds_read_b64_tr_b4.
#include <algorithm>

#include "cache_ops.h"
#include "row_device.h"

namespace tts {

namespace {

using row_ops::Dwords;
using row_ops::f16x8;
using row_ops::f32x4;
using row_ops::load_dwords;
using row_ops::mfma16;
using row_ops::u32;

constexpr int WAVES = 4, BLOCK = 64;  // tokens
constexpr float LOG2_E = 1.4426950408889634f;

typedef int i32x2 __attribute__((ext_vector_type(2)));

// f over the four lanes of a row (those 16 apart)
template <class F>
__device__ __forceinline__ float over_row(float v, F f) {
  v = f(v, __shfl_xor(v, 16));
  return f(v, __shfl_xor(v, 32));
}

// a word's codes as four pairs, in the order of its bits 0 and 16, 4 and 20, 8 and 24, 12 and 28; the second and the last 2^4 as much
__device__ __forceinline__ uint4 codes_of(u32 w) { return make_uint4(w & 0x000f000fu, w & 0x00f000f0u, w >> 8 & 0x000f000fu, w >> 8 & 0x00f000f0u); }

__device__ __forceinline__ float half_of(u32 pair, bool bf16, bool upper) {
  if (bf16) return __uint_as_float(upper ? pair & 0xffff0000u : pair << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(upper ? pair >> 16 : pair));
}

__device__ __forceinline__ u32 fp16_pair(float a, float b) {
  const tts_gemm_device::f16x2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(u32, v);
}

// The request and the rows of it that a workgroup has; what follows of them for tokens.
struct Rows {
  int request, first, rows;       // of the step's rows: where the request's begin, and how many it has
  int length, tokens;             // of the request, and how many of them the table can hold
  int begin, end;                 // what the tile's rows see lies in [begin, end), begin at a multiple of 16
  int slices;
};

// (starts are the caller's memory: whatever they hold, rows stay inside [0, tokens))
__device__ __forceinline__ int start_of(const AttendParams &p, int b) { return (int)min((int64_t)max(p.starts[b], 0), p.tokens); }

__device__ __forceinline__ Rows rows_of(const AttendParams &p, int b, int tile) {
  Rows r;
  r.request = b, r.first = start_of(p, b), r.rows = max(start_of(p, b + 1) - r.first, 0);
  r.length = max(p.lengths[b], 0);
  r.tokens = (int)min((int64_t)r.length, (int64_t)p.columns * p.cache.page);
  const int top = tile * p.plan.tile / p.group, bottom = min((tile * p.plan.tile + p.plan.tile - 1) / p.group, r.rows - 1);
  const int behind = r.length - r.rows + 1;  // what row 0 sees ends there
  r.begin = p.window ? max(behind + top - p.window, 0) / 16 * 16 : 0;
  r.end = min(behind + bottom, r.tokens);
  const int slices = (r.end - r.begin + p.plan.slice - 1) / p.plan.slice;
  r.slices = min(max(slices, 1), p.plan.slices);
  return r;
}

// W: dim / 32.  RT: tiles of 16 rows per wavefront.  BY_ROWS: wavefronts have rows of their own; else all have the same rows, and blocks in turn.
template <bool BF16, int W, int RT, bool BY_ROWS>
__global__ __launch_bounds__(256) void kv4_attend_kernel(AttendParams p) {
  constexpr int D = 32 * W, PITCH = D / 2 + 8, V_BYTES = BLOCK * PITCH, WAVE_BYTES = V_BYTES + 2 * 4 * BLOCK, TILE = BY_ROWS ? WAVES * RT * 16 : RT * 16;
  constexpr int MEET_BYTES = BY_ROWS ? 0 : (WAVES / 2) * RT * 16 * (D + 2) * 4;
  __shared__ __attribute__((aligned(16))) char lds[MEET_BYTES > WAVES * WAVE_BYTES ? MEET_BYTES : WAVES * WAVE_BYTES];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), m = lane % 16, g = lane / 16;
  const int kv_heads = p.cache.heads, item = blockIdx.x / kv_heads, kv = blockIdx.x % kv_heads, slice = blockIdx.y;

  if (p.clear && kv == 0 && slice == 0) {  // rows of no request
    const int64_t from = p.requests ? start_of(p, 0) : 0, to = p.requests ? start_of(p, p.requests) : 0, others = from + p.tokens - max(from, to), size = (int64_t)p.heads * D;
    for (int64_t i = item; i < others; i += p.plan.items) {
      uint16_t *row = (uint16_t *)p.out + (i < from ? i : max(from, to) + i - from) * p.o_token;
      for (int64_t e = threadIdx.x; e < size; e += 256) row[e / D * p.o_head + e % D] = 0;
    }
  }
  if (!p.requests) return;

  // Tiles of request b are numbered from floor(starts[b] * group / TILE) + b: that leaves room for all of them, whatever the requests before have
  int b = -1;
  for (int at = 0; at < p.requests; at += 64) {
    const bool before = at + lane < p.requests && (int)((int64_t)start_of(p, min(at + lane, p.requests - 1)) * p.group / TILE) + at + lane <= item;
    b += __popcll(__ballot(before));
  }
  b = max(b, 0);
  const int tile = item - (int)((int64_t)start_of(p, b) * p.group / TILE) - b;
  const Rows r = rows_of(p, b, tile);
  if (tile < 0 || (int64_t)tile * TILE >= (int64_t)r.rows * p.group || slice >= r.slices) return;

  char *const mine = lds + wave * WAVE_BYTES;
  u32 *const key_pairs = (u32 *)(mine + V_BYTES), *const value_pairs = key_pairs + BLOCK;
  const int row0 = tile * TILE + (BY_ROWS ? wave * RT * 16 : 0);  // of the request's tokens and the group's heads

  // The rows: what they see, and q as operands
  int low[RT], high[RT];  // [low, high)
  int64_t row_at[RT];     // token * heads + head, -1: no row
  float factor[RT], sum_q[RT];
  uint4 q[RT][W];
  for (int t = 0; t < RT; t++) {
    const int row = row0 + t * 16 + m, token = row / p.group, head = kv * p.group + row % p.group;
    const bool live = token < r.rows;
    row_at[t] = live ? (int64_t)(r.first + token) * p.heads + head : -1;
    const int position = r.length - r.rows + token;
    low[t] = p.window ? max(position - p.window + 1, 0) : 0;
    high[t] = live ? min(position + 1, r.tokens) : 0;
    float v[W][8], most = 0.f, sum = 0.f;
    const char *from = (const char *)p.q + 2 * ((int64_t)(r.first + (live ? token : 0)) * p.q_token + (int64_t)head * p.q_head) + 16 * g * W;
    for (int w = 0; w < W; w++) {
      const Dwords<4> x = load_dwords<4>(from + 16 * w);
      for (int e = 0; e < 8; e++) {
        v[w][e] = live ? half_of(x.d[e / 2], BF16, e & 1) : 0.f;
        most = fmaxf(most, fabsf(v[w][e])), sum += v[w][e];
      }
    }
    most = over_row(most, [](float a, float b) { return fmaxf(a, b); });
    sum = over_row(sum, [](float a, float b) { return a + b; });
    const float scaled = row_ops::fp16_scale(most);
    for (int w = 0; w < W; w++) {
      float x[8];
      for (int e = 0; e < 8; e++) x[e] = v[w][e] * (e & 2 ? scaled * 0x1p-4f : scaled);
      q[t][w] = make_uint4(fp16_pair(x[0], x[1]), fp16_pair(x[2], x[3]), fp16_pair(x[4], x[5]), fp16_pair(x[6], x[7]));
    }
    factor[t] = p.scale * LOG2_E * 0x1p24f / scaled;
    // (a row with an infinity: NaN, as the formula gives, also where all its scores are -inf here)
    sum_q[t] = (sum - sum == 0.f ? sum : __builtin_nanf("")) * p.scale * LOG2_E;
  }

  // all of a block's tokens are seen by all of the wavefront's rows where it lies inside [seen_from, seen_to)
  int seen_from, seen_to, last;
  {
    const int top = row0 / p.group, bottom = min((row0 + RT * 16 - 1) / p.group, r.rows - 1), behind = r.length - r.rows + 1;
    seen_from = p.window ? max(behind + bottom - p.window, 0) : 0;
    seen_to = min(behind + top, r.tokens);
    last = top < r.rows ? min(behind + bottom, r.tokens) : 0;
  }
  const int begin = r.begin + slice * p.plan.slice, end = min(slice == r.slices - 1 ? r.end : begin + p.plan.slice, last);
  constexpr int STEP = BY_ROWS ? BLOCK : WAVES * BLOCK;
  const int start = begin + (BY_ROWS ? 0 : wave * BLOCK);
  const int blocks = end > start ? (end - start + STEP - 1) / STEP : 0;

  const char *const cache = (const char *)p.cache.base + (int64_t)kv * p.cache.head_bytes;
  const int page = p.cache.page;
  f32x4 out[D / 16][RT];
  float top[RT], total[RT], lowest[RT];
  for (int t = 0; t < RT; t++) {
    top[t] = -__builtin_inff(), total[t] = 0.f, lowest[t] = 0.f;
    for (int d = 0; d < D / 16; d++) out[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int power = -112;  // values' steps are below 2^power

  // the table's entries of 16 blocks: lane 4 n + j has that of tile j of block n
  int entry = 0, within = 0;
  unsigned long long there = 0;
  auto look_up = [&](int n) __attribute__((always_inline)) {
    const int token = start + (n + lane / 4) * STEP + lane % 4 * 16, column = token / page;
    entry = -1;
    if (token < end) entry = p.table[(int64_t)r.request * p.ld_table + column];  // (end is inside the table)
    const bool ok = entry >= 0 && entry < p.cache.pages;
    there = __ballot(ok);
    entry = ok ? entry : 0, within = token % page;
  };
  struct Block {
    Dwords<W> k[4], v[4];
    u32 kp, vp;
  };
  auto load_block = [&](int n) __attribute__((always_inline)) {
    Block x;
    for (int j = 0; j < 4; j++) {
      const int at = n % 16 * 4 + j;
      const int64_t of = (int64_t)__builtin_amdgcn_readlane(entry, at) * p.cache.page_bytes + (int64_t)__builtin_amdgcn_readlane(within, at) * (D / 2);
      const char *codes = cache + of + m * (D / 2) + g * (4 * W);
      x.k[j] = load_dwords<W>(codes), x.v[j] = load_dwords<W>(codes + (int64_t)page * (D / 2));
    }
    const int at = n % 16 * 4 + g, token = start + n * STEP + lane;
    const char *pairs = cache + (int64_t)__shfl(entry, at) * p.cache.page_bytes + (int64_t)page * D + (__shfl(within, at) + m) * 4;
    x.kp = *(const u32 *)pairs, x.vp = *(const u32 *)(pairs + page * 4);
    if (token >= end || !(there >> at & 1)) x.kp = x.vp = 0;  // (memory that was never written may hold any)
    return x;
  };

  for (int n = 0; n < blocks; n++) {
    if (n % 16 == 0) look_up(n);
    const Block x = load_block(n);
    // values and pairs to LDS: the 16 tokens of a lane's operand in a row, 8 bytes between rows
    for (int j = 0; j < 4; j++) __builtin_memcpy(mine + (m / 4 * 16 + j * 4 + m % 4) * PITCH + g * (4 * W), &x.v[j], 4 * W);
    key_pairs[lane] = x.kp, value_pairs[lane] = x.vp;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x4 s[4][RT];
    for (int j = 0; j < 4; j++) {
      for (int t = 0; t < RT; t++) s[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < W; w++) {
        const uint4 k = codes_of(x.k[j].d[w]);
        for (int t = 0; t < RT; t++) s[j][t] = mfma16<false>(k, q[t][w], s[j][t]);
      }
    }
    float value_step[4][4], value_low[4][4], most_step = 0.f;
    for (int j = 0; j < 4; j++) {
      const uint4 kp = *(const uint4 *)(key_pairs + 16 * j + 4 * g), vp = *(const uint4 *)(value_pairs + 16 * j + 4 * g);
      const u32 k[4] = {kp.x, kp.y, kp.z, kp.w}, v[4] = {vp.x, vp.y, vp.z, vp.w};
      for (int i = 0; i < 4; i++) {
        const float step = half_of(k[i], BF16, false), low_k = half_of(k[i], BF16, true);
        for (int t = 0; t < RT; t++) s[j][t][i] = s[j][t][i] * factor[t] * step + low_k * sum_q[t];
        value_step[j][i] = half_of(v[i], BF16, false), value_low[j][i] = half_of(v[i], BF16, true);
        most_step = fmaxf(most_step, value_step[j][i]);
      }
    }
    const int first = start + n * STEP;
    const bool whole = first >= seen_from && first + BLOCK <= seen_to && (there >> (n % 16 * 4) & 15) == 15;
    u32 seen[RT];
    for (int t = 0; t < RT; t++) seen[t] = 0xffff;
    if (!whole)
      for (int t = 0; t < RT; t++) {
        seen[t] = 0;
        for (int j = 0; j < 4; j++)
          for (int i = 0; i < 4; i++) {
            const int token = first + 16 * j + 4 * g + i;
            const bool ok = token >= low[t] && token < min(high[t], end) && (there >> (n % 16 * 4 + j) & 1);
            seen[t] |= (u32)ok << (4 * j + i);
            s[j][t][i] = ok ? s[j][t][i] : -__builtin_inff();
          }
      }
    most_step = over_row(most_step, [](float a, float b) { return fmaxf(a, b); });
    const int power_now = most_step > 0.f && most_step < __builtin_inff() ? max(power, __builtin_amdgcn_frexp_expf(most_step)) : power;
    const float unit = __builtin_amdgcn_ldexpf(1.f, 14 - power_now);
    for (int j = 0; j < 4; j++)
      for (int i = 0; i < 4; i++) value_step[j][i] *= unit * (i & 1 ? 0x1p-4f : 1.f);
    uint4 weights[2][RT];
    for (int t = 0; t < RT; t++) {
      float most = -__builtin_inff();
      for (int j = 0; j < 4; j++)
        for (int i = 0; i < 4; i++) most = fmaxf(most, s[j][t][i]);
      most = fmaxf(top[t], over_row(most, [](float a, float b) { return fmaxf(a, b); }));
      const float from = most == -__builtin_inff() ? 0.f : most;  // (nothing seen yet)
      const float kept = __builtin_amdgcn_exp2f(top[t] - from);
      top[t] = most;
      total[t] *= kept, lowest[t] *= kept;
      const float moved = __builtin_amdgcn_ldexpf(kept, power - power_now);
      for (int d = 0; d < D / 16; d++)
        for (int i = 0; i < 4; i++) out[d][t][i] *= moved;
      float weight[4][4];
      for (int j = 0; j < 4; j++)
        for (int i = 0; i < 4; i++) {
          const bool ok = seen[t] >> (4 * j + i) & 1;
          const float e = __builtin_amdgcn_exp2f(s[j][t][i] - from);
          total[t] += e;
          // (a step or lowest value of NaN stays with the rows that see it)
          lowest[t] += ok ? e * value_low[j][i] : 0.f;
          weight[j][i] = ok ? e * value_step[j][i] : 0.f;
        }
      for (int h = 0; h < 2; h++)
        weights[h][t] = make_uint4(fp16_pair(weight[2 * h][0], weight[2 * h + 1][0]), fp16_pair(weight[2 * h][1], weight[2 * h + 1][1]), fp16_pair(weight[2 * h][2], weight[2 * h + 1][2]),
                                   fp16_pair(weight[2 * h][3], weight[2 * h + 1][3]));
    }
    power = power_now;
    for (int d = 0; d < D / 16; d++) {
      const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32((i32x2 __attribute__((address_space(3))) *)((__attribute__((address_space(3))) void *)(mine + lane * PITCH + 8 * d)));
      const uint4 first_half = codes_of(v[0]), second_half = codes_of(v[1]);
      for (int t = 0; t < RT; t++) out[d][t] = mfma16<false>(first_half, weights[0][t], out[d][t]);
      for (int t = 0; t < RT; t++) out[d][t] = mfma16<false>(second_half, weights[1][t], out[d][t]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  for (int t = 0; t < RT; t++) {
    const auto add = [](float a, float b) { return a + b; };
    total[t] = over_row(total[t], add), lowest[t] = over_row(lowest[t], add);
    for (int d = 0; d < D / 16; d++)
      for (int i = 0; i < 4; i++) out[d][t][i] = __builtin_amdgcn_ldexpf(out[d][t][i], 10 + power) + lowest[t];
  }
  if constexpr (!BY_ROWS) {  // the wavefronts' parts, two to two and one to one
    constexpr int PART = RT * 16 * (D + 2) * 4;
    for (int half = WAVES / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        float *to = (float *)(lds + (wave - half) * PART);
        for (int t = 0; t < RT; t++) {
          for (int d = 0; d < D / 16; d++) *(f32x4 *)(to + (t * (D / 16) + d) * 256 + lane * 4) = out[d][t];
          if (g == 0) to[RT * 16 * D + t * 16 + m] = top[t], to[RT * 16 * D + RT * 16 + t * 16 + m] = total[t];
        }
      }
      __syncthreads();
      if (wave < half) {
        const float *from = (const float *)(lds + wave * PART);
        for (int t = 0; t < RT; t++) {
          const float other = from[RT * 16 * D + t * 16 + m], more = from[RT * 16 * D + RT * 16 + t * 16 + m];
          const float most = fmaxf(top[t], other), base = most == -__builtin_inff() ? 0.f : most;
          const float here = __builtin_amdgcn_exp2f(top[t] - base), there_too = __builtin_amdgcn_exp2f(other - base);
          top[t] = most, total[t] = total[t] * here + more * there_too;
          for (int d = 0; d < D / 16; d++) {
            const f32x4 add = *(const f32x4 *)(from + (t * (D / 16) + d) * 256 + lane * 4);
            for (int i = 0; i < 4; i++) out[d][t][i] = out[d][t][i] * here + add[i] * there_too;
          }
        }
      }
    }
    if (wave != 0) return;
  }
  for (int t = 0; t < RT; t++) {
    if (row_at[t] < 0) continue;
    if (r.slices == 1) {
      const float over = total[t] == 0.f ? 0.f : 1.f / total[t];  // (a row that sees nothing: zeros)
      const int64_t token = row_at[t] / p.heads, head = row_at[t] % p.heads;
      char *to = (char *)p.out + 2 * (token * p.o_token + head * p.o_head) + 8 * g;
      for (int d = 0; d < D / 16; d++) {
        u32 w[2];
        for (int i = 0; i < 2; i++) {
          const float a = out[d][t][2 * i] * over, c = out[d][t][2 * i + 1] * over;
          w[i] = BF16 ? (u32)__builtin_bit_cast(uint16_t, (__bf16)a) | (u32)__builtin_bit_cast(uint16_t, (__bf16)c) << 16 : fp16_pair(a, c);
        }
        __builtin_memcpy(to + 32 * d, w, 8);
      }
    } else {
      const int64_t part = row_at[t] * p.plan.slices + slice;
      for (int d = 0; d < D / 16; d++) *(f32x4 *)(p.parts + part * D + 16 * d + 4 * g) = out[d][t];
      if (g == 0) p.stats[part * 2] = top[t], p.stats[part * 2 + 1] = total[t];
    }
  }
}

// The slices of a row, where there are several: a wavefront per row, in the order of the slices.
template <bool BF16>
__global__ __launch_bounds__(256) void kv4_attend_join_kernel(AttendParams p) {
  const int lane = threadIdx.x % 64, dim = p.cache.dim;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64, token = row / p.heads;
  if (token >= p.tokens) return;
  const int head = (int)(row % p.heads);
  int b = -1;
  for (int at = 0; at < p.requests; at += 64) b += __popcll(__ballot(at + lane < p.requests && start_of(p, min(at + lane, p.requests - 1)) <= token));
  if (b < 0) return;
  const int first = start_of(p, b);
  if (token >= start_of(p, b + 1)) return;  // (a row of no request)
  const Rows r = rows_of(p, b, (int)(((token - first) * p.group + head % p.group) / p.plan.tile));
  if (r.slices == 1) return;  // (written already)
  const float *stats = p.stats + row * p.plan.slices * 2, *parts = p.parts + row * p.plan.slices * dim;
  float most = -__builtin_inff();
  for (int i = 0; i < r.slices; i++) most = fmaxf(most, stats[2 * i]);
  const float base = most == -__builtin_inff() ? 0.f : most;
  float total = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < r.slices; i++) {
    const float share = __builtin_amdgcn_exp2f(stats[2 * i] - base);
    total += stats[2 * i + 1] * share;
    for (int n = 0; n < 4; n++)
      if (lane + 64 * n < dim) sum[n] += parts[(int64_t)i * dim + lane + 64 * n] * share;
  }
  const float over = total == 0.f ? 0.f : 1.f / total;
  uint16_t *to = (uint16_t *)p.out + token * p.o_token + head * p.o_head;
  for (int n = 0; n < 4; n++)
    if (lane + 64 * n < dim) to[lane + 64 * n] = BF16 ? __builtin_bit_cast(uint16_t, (__bf16)(sum[n] * over)) : __builtin_bit_cast(uint16_t, (_Float16)(sum[n] * over));
}

template <bool BF16, int W>
hipError_t launch_of(const AttendParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.plan.items * p.cache.heads), (unsigned)p.plan.slices);
  if (p.plan.by_rows) kv4_attend_kernel<BF16, W, 2, true><<<grid, 256, 0, s>>>(p);
  else if (p.plan.row_tiles == 2) kv4_attend_kernel<BF16, W, 2, false><<<grid, 256, 0, s>>>(p);
  else kv4_attend_kernel<BF16, W, 1, false><<<grid, 256, 0, s>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.plan.slices > 1) {
    kv4_attend_join_kernel<BF16><<<dim3((unsigned)((p.tokens * p.heads + 3) / 4)), 256, 0, s>>>(p);
    e = hipGetLastError();
  }
  return e;
}

template <bool BF16>
hipError_t launch_as(const AttendParams &p, hipStream_t s) {
  switch (p.cache.dim / 32) {
    case 1: return launch_of<BF16, 1>(p, s);
    case 2: return launch_of<BF16, 2>(p, s);
    case 3: return launch_of<BF16, 3>(p, s);
    case 4: return launch_of<BF16, 4>(p, s);
    case 5: return launch_of<BF16, 5>(p, s);
    case 6: return launch_of<BF16, 6>(p, s);
    case 7: return launch_of<BF16, 7>(p, s);
    default: return launch_of<BF16, 8>(p, s);
  }
}

}  // namespace

AttendPlan plan_attend(int64_t tokens, int requests, int heads, int kv_heads, int dim, int64_t longest, int window) {
  AttendPlan plan = {};
  const int64_t group = heads / kv_heads, rows = (tokens + requests - 1) / std::max(requests, 1) * group;  // of a request, on average
  plan.by_rows = rows > 64;
  plan.row_tiles = rows > 16 ? 2 : 1;
  plan.tile = plan.by_rows ? WAVES * plan.row_tiles * 16 : plan.row_tiles * 16;
  plan.items = std::max<int64_t>(1, tokens * group / plan.tile + requests);
  const int64_t range = window ? std::min<int64_t>(longest, (int64_t)window + plan.tile / group + 17) : longest;
  const int64_t groups = std::max<int64_t>(1, plan.items * kv_heads), wanted = 1024;
  const int64_t least = WAVES * BLOCK;  // tokens of a slice
  int64_t slices = std::max<int64_t>(1, std::min((wanted + groups - 1) / groups, (range + least - 1) / least));
  plan.slice = (int)std::max<int64_t>(((range + slices - 1) / slices + least - 1) / least * least, least);
  plan.slices = (int)std::max<int64_t>(1, (range + plan.slice - 1) / plan.slice);
  return plan;
}

size_t attend_workspace_bytes(const AttendPlan &plan, int64_t tokens, int heads, int dim) {
  return plan.slices > 1 ? (size_t)tokens * heads * plan.slices * (dim + 2) * sizeof(float) : 0;
}

hipError_t launch_attend(const AttendParams &p, hipStream_t s) { return p.cache.bf16 ? launch_as<true>(p, s) : launch_as<false>(p, s); }

}  // namespace tts
