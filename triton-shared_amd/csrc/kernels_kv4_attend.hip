// Attention over the paged cache held in 4 bits (its layout: cache_ops.h).  Of a row (a token and a head) at position i of a request:
//   s_j = scale * q . k_j over the tokens j it sees (i - window < j <= i, in a page that the table has),  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).
// With k_j = a_j c_j + b_j and v_j = a'_j c'_j + b'_j (codes c of 0 .. 15, a step a and a lowest value b of the token's head):
//   s_j = scale * (a_j (q . c_j) + b_j sum(q)),   out = (sum_j (p_j a'_j) c'_j + sum_j p_j b'_j) / sum_j p_j,
// so the matrix instructions multiply codes.  A code in bits 0 .. 3 or 4 .. 7 of a half is the fp16 c 2^-24 or c 2^-20 (a number below the normal
// ones, which they take as it is): eight codes of a 32-bit word become four pairs with four ands and one shift, and what is multiplied with the second kind is
// 2^-4 of itself.  q goes in as fp16 times a power of two per row that takes its largest element to [2^13, 2^14): exactly, but for 2^-34 of that element.
// p_j a'_j goes in as fp16, times a power of two per row that takes the largest a' that it has seen so far to [2^13, 2^14) and 2^-4 for every second token: within 2^-11 of it, less than the rounding of a
// bf16 output (2^-8); where the output is fp16 too, as the sum of two (2^-22); and within 2^-34 of the largest a'.  All sums and the statistics are in 32 bits.
// (The sum of two for bf16 as well: 64 ragged requests 36.5 us (one 35.3), 5 tokens each of 16 requests 30.4 (25.7), prompts, as fp16 has them, 258 (221),
// for errors against the exact result of 1.71e-3 instead of 1.73e-3, of which 1.71e-3 is the output's rounding.)
//
// A wavefront takes blocks of 64 tokens.  Keys: lane (m, g) = (lane % 16, lane / 16) loads a quarter g of token m of each of four tiles, which is the
// left operand of  scores[token][row];  so a lane gets the scores of tokens 4 g .. 4 g + 3 of each tile for row m, and what it makes of them is the right
// operand of  out[element][row]  as it stands.  Its left operand, 16 tokens of one element per lane, is read out of LDS by ds_read_b64_tr_b4.
//
// What bounds it, dim 128 and 8 heads of the cache, bf16 (a copy of 1 GiB runs at 5.0 TB/s, a 16-bit matrix product of 8192^3 at 1.19 PFLOP/s):
//   64 requests of 100 .. 8192 tokens (118 MB): 35 us in a graph, of which joining the slices 4: 3.8 TB/s while it runs.  The chain before a workgroup's first block, 3.4 us where it is alone
//     (lengths, table and codes, one after another), and its last steps are not hidden by others: there is one round of workgroups, and more of them cost as much as they hide.
//   2 of 131072, 64 heads of q: 35 us, 29 + 6: 4.4 TB/s.   1 of 4000: 11.8 us, 8.5 + 3.3: the chains.
//   4 x 1024 rows behind up to 4096 tokens: 221 us, 598 TFLOP/s (of an fp16 cache 258, 512): the vector instructions, some 570 to 64 matrix instructions in a block of 32 rows (160 of them unpack codes, 350 are the softmax); they
//     fill two thirds of the cycles, the matrix instructions a quarter, and two wavefronts per SIMD, which is what 234 registers allow, hide little of one behind the other.
#include <algorithm>
#include <type_traits>

#include "cache_ops.h"
#include "lanes.h"
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
constexpr int MOST_SLICES = 128;
constexpr float LOG2_E = 1.4426950408889634f;

typedef int i32x2 __attribute__((ext_vector_type(2)));

// f over the lanes of a row: those 16 apart by exchanges of 16 and of 32 lanes in registers, and those ROWS apart in 16 lanes
template <int ROWS = 16, class F>
__device__ __forceinline__ float over_row(float v, F f) {
  if constexpr (ROWS <= 4) v = f(v, dpp_moved<0x124>(v));  // row_ror 4
  if constexpr (ROWS <= 8) v = f(v, dpp_moved<0x128>(v));
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
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

// What a call's workgroups (of one head of the cache) do: each request's tiles of rows, one after another, and of each its slices of the tokens that the request's
// rows see.  Slices are of one length for all requests, so that a batch of ragged lengths makes workgroups of one size: their number is what the call has beyond one for each
// tile, and their length what it takes to deal all tokens to that many.  Every wavefront works that out for itself, a request per lane.
struct Work {
  int request, first, rows;     // of the step's rows: where the request's begin, and how many it has (0: nothing to do)
  int tile, slice, slices;
  int length, tokens;           // up to the last of these rows, and how many of them the table can hold
  int begin, size;              // the first token that its rows see, at a multiple of 16, and a slice's tokens
  int index;                    // of its first workgroup
};

// (starts are the caller's memory: whatever they hold, rows stay inside [0, tokens))
__device__ __forceinline__ int start_of(const AttendParams &p, int b) { return (int)min((int64_t)max(p.starts[b], 0), p.tokens); }

// at - by, at least 0 (`at` may be negative, and the difference none of 32 bits)
__device__ __forceinline__ int behind(int at, int by) { return max(at, by) - by; }

struct Request {
  int first, rows, length, tokens, begin, blocks, tiles;  // blocks: of 64 tokens, of what its rows see
};
__device__ __forceinline__ Request request_of(const AttendParams &p, int b) {
  Request r = {};
  if (b >= p.requests) return r;
  r.first = start_of(p, b);
  const int next = start_of(p, b + 1), length = p.lengths[b];
  // (of more new tokens than q has rows the first have one, and what lies behind them is none of theirs to see; far below 0 nothing changes any more)
  r.rows = max(next - r.first, 0), r.length = max(max(length, 0) - (max(p.starts[b + 1], 0) - next), -(1 << 30));
  r.tokens = min(max(r.length, 0), p.places);
  r.begin = p.window ? min(behind(r.length - r.rows + 1, p.window), r.tokens) & ~15 : 0;  // (at most places: what is added to it stays in 32 bits)
  r.blocks = (max(r.tokens - r.begin, 0) + BLOCK - 1) / BLOCK;
  r.tiles = (r.rows * p.group + (1 << p.plan.tile_log) - 1) >> p.plan.tile_log;
  return r;
}

// the sum of v over the lanes up to this one
__device__ __forceinline__ int sum_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: a row's last to the next one
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: the first half's to the second
  return v;
}

// the work of workgroup `index`; or of the request that holds row `row` of the step, with `index` < 0
__device__ __forceinline__ Work work_of(const AttendParams &p, int index, int row) {
  const int lane = threadIdx.x % 64, tile_log = p.plan.tile_log;
  Request r = request_of(p, lane);
  int size = 1 << 24;  // of a slice, in blocks: all
  if (p.plan.extra) {
    float all = (float)r.tiles * (float)r.blocks;
    int most = r.blocks;
    for (int at = 64; at < p.requests; at += 64) {
      const Request o = request_of(p, at + lane);
      all += (float)o.tiles * (float)o.blocks, most = max(most, o.blocks);
    }
    all = over_lanes<16>(all, [](float a, float b) { return a + b; }), all = over_row(all, [](float a, float b) { return a + b; });
    const float longest = over_lanes<16>((float)most, [](float a, float b) { return fmaxf(a, b); });
    // (rounded up past what 32 bits lose: no more slices than there are workgroups)
    const float each = fmaxf(all * p.plan.over_extra * 1.0001f, over_row(longest, [](float a, float b) { return fmaxf(a, b); }) * (1.0001f / MOST_SLICES));
    size = ((int)fminf(each, 16777000.f) + WAVES) / WAVES * WAVES;
  }
  Work w = {};
  int before = 0;
  for (int at = 0; at < p.requests; at += 64) {
    if (at) r = request_of(p, at + lane);
    const int slices = r.blocks > size ? (int)((u32)(r.blocks + size - 1) / (u32)size) : 1, count = r.tiles * slices, upto = sum_upto(count);
    const bool here = index < 0 ? row >= r.first && row < r.first + r.rows : index >= before + upto - count && index < before + upto;
    const unsigned long long found = __ballot(here);
    if (found) {
      const int at_lane = __builtin_ctzll(found);
      auto get = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, at_lane); };
      w.request = at + at_lane, w.first = get(r.first), w.rows = get(r.rows), w.length = get(r.length), w.tokens = get(r.tokens), w.begin = get(r.begin);
      w.slices = get(slices), w.index = before + get(upto - count);
      w.size = size * BLOCK;
      if (w.slices > 1) {  // slices of one length within the request
        const u32 blocks = (u32)get(r.blocks);
        w.size = (int)(((blocks + w.slices - 1) / (u32)w.slices + WAVES - 1) / WAVES * WAVES) * BLOCK;
      }
      const int of = index - w.index;
      w.tile = index < 0 ? ((row - w.first) * p.group) >> tile_log : w.slices > 1 ? (int)((u32)of / (u32)w.slices) : of;
      w.slice = index < 0 ? 0 : of - w.tile * w.slices;
      // (only where starts are not in order may it not have that tile, or workgroup)
      if (w.tile < 0 || w.tile >= get(r.tiles) || w.slice < 0 || w.index < 0 || (int64_t)w.index + (int64_t)(w.tile + 1) * w.slices > p.plan.items + p.plan.extra) w.rows = 0;
      return w;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return w;
}

// of a wavefront that has rows of its own: what the registers of two wavefronts per SIMD hold
constexpr int row_tiles_of(int w) { return w <= 4 ? 2 : 1; }

// W: dim / 32.  RT: tiles of rows per wavefront, ROWS: of such a tile.  OWN: what of a workgroup's wavefronts have of their own: blocks of tokens, in turn; rows; heads of the cache.
// The matrix instructions' tiles have 16 rows.  Of fewer (a token's heads of one key's) each is there 16 / ROWS times, and of the scores that a lane gets so, those of 4
// tiles of tokens, it goes on with 4 ROWS / 16 of them: the copies share the softmax.
template <bool BF16, int W, int RT, int ROWS, int OWN>
__global__ __launch_bounds__(256, W > 4 || OWN == OWN_ROWS || (!BF16 && W == 4 && ROWS == 16) ? 2 : 3) void kv4_attend_kernel(AttendParams p) {
  constexpr int D = 32 * W, PITCH = D / 2 + 8, V_BYTES = BLOCK * PITCH, WAVE_ROWS = RT * ROWS, WAVE_BYTES = V_BYTES + 4 * 4 * BLOCK + 4 * 2 * WAVE_ROWS, TILE = (OWN == OWN_ROWS ? WAVES : 1) * WAVE_ROWS;
  constexpr int BANKS = 16 / ROWS, NJ = 4 / BANKS;
  constexpr int MEET_PITCH = D + 4, MEET_BYTES = OWN != OWN_BLOCKS ? 0 : WAVES * WAVE_ROWS * (MEET_PITCH + 2) * 4;
  __shared__ __attribute__((aligned(16))) char lds[MEET_BYTES > WAVES * WAVE_BYTES ? MEET_BYTES : WAVES * WAVE_BYTES];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), m = lane % 16, g = lane / 16, bank = m / ROWS;
  const int kv_heads = p.cache.heads, per_item = OWN == OWN_HEADS ? (kv_heads + WAVES - 1) / WAVES : kv_heads, groups = (int)(p.plan.items + p.plan.extra) * per_item;

  if ((int)blockIdx.x >= groups) {  // rows of no request
    const int64_t from = p.requests ? start_of(p, 0) : 0, to = max(from, p.requests ? (int64_t)start_of(p, p.requests) : 0), others = from + p.tokens - to, size = (int64_t)p.heads * D;
    for (int64_t i = blockIdx.x - groups; i < others; i += gridDim.x - groups) {
      uint16_t *row = (uint16_t *)p.out + (i < from ? i : to + i - from) * p.o_token;
      for (int64_t e = threadIdx.x; e < size; e += 256) row[e / D * p.o_head + e % D] = 0;
    }
    return;
  }
  // (the last first: of a prompt's tiles those have the most tokens)
  const int behind_it = divided(blockIdx.x, p.by_per_item), item = (int)(p.plan.items + p.plan.extra) - 1 - behind_it;
  const int kv = OWN == OWN_HEADS ? (int)(blockIdx.x - behind_it * per_item) * WAVES + wave : blockIdx.x - behind_it * per_item;
  const Work r = work_of(p, item, 0);
  if (!r.rows || (OWN == OWN_HEADS && kv >= kv_heads)) return;

  char *const mine = lds + wave * WAVE_BYTES;
  float *const key_step = (float *)(mine + V_BYTES), *const key_low = key_step + BLOCK, *const value_step = key_low + BLOCK, *const value_low = value_step + BLOCK;
  float *const lifts = value_low + BLOCK;            // of the rows
  int *const powers = (int *)(lifts + WAVE_ROWS);  // ... values' steps that it has seen are up to 2^power
  const int row0 = r.tile * TILE + (OWN == OWN_ROWS ? wave * WAVE_ROWS : 0);  // of the request's tokens and the group's heads

  // The rows, what they see, and q, on its way
  int low[RT], high[RT];  // [low, high)
  Dwords<4> raw[RT][W];
  for (int t = 0; t < RT; t++) {
    const int row = row0 + t * ROWS + m % ROWS, token = divided(row, p.by_group), head = kv * p.group + row - token * p.group;
    const bool live = token < r.rows;
    const int position = r.length - r.rows + token;
    low[t] = p.window ? behind(position, p.window - 1) : 0;
    high[t] = live ? min(position + 1, r.tokens) : 0;
    const char *from = (const char *)p.q + 2 * ((int64_t)(r.first + (live ? token : 0)) * p.q_token + (int64_t)head * p.q_head) + 16 * g * W;
    for (int w = 0; w < W; w++) raw[t][w] = load_dwords<4>(from + 16 * w);
  }

  // all of a block's tokens are seen by all of the wavefront's rows where it lies inside [seen_from, seen_to)
  int seen_from, seen_to, last, window_begin;  // (the last two: where what any of them sees ends, and begins, at a multiple of 16)
  {
    const int top = divided(row0, p.by_group), bottom = min(divided(row0 + WAVE_ROWS - 1, p.by_group), r.rows - 1), sees = r.length - r.rows + 1;  // (row 0: up to there)
    seen_from = p.window ? behind(sees + bottom, p.window) : 0;
    seen_to = min(sees + top, r.tokens);
    last = top < r.rows ? min(sees + bottom, r.tokens) : 0;
    window_begin = p.window ? min(behind(sees + top, p.window), r.tokens) & ~15 : 0;
  }
  const int slice_begin = r.begin + r.slice * r.size, end = __builtin_amdgcn_readfirstlane(min(slice_begin + r.size, last)), begin = max(slice_begin, window_begin);
  seen_from = __builtin_amdgcn_readfirstlane(seen_from), seen_to = __builtin_amdgcn_readfirstlane(min(seen_to, end));
  constexpr int STEP = OWN != OWN_BLOCKS ? BLOCK : WAVES * BLOCK;
  const int start = __builtin_amdgcn_readfirstlane(begin + (OWN != OWN_BLOCKS ? 0 : wave * BLOCK));
  const int blocks = __builtin_amdgcn_readfirstlane(end > start ? (end - start + STEP - 1) / STEP : 0);

  const char *const cache = (const char *)p.cache.base + (int64_t)kv * p.cache.head_bytes;
  const int page = p.cache.page;
  // where the tiles of 16 blocks are in the cache: lane 4 n + j has tile j of block n
  int64_t codes_at = 0, pairs_at = 0;
  unsigned long long there = 0;
  auto look_up = [&](int n) __attribute__((always_inline)) {
    const int token = start + (n + lane / 4) * STEP + lane % 4 * 16, column = divided(token, p.cache.by_page);
    int entry = -1;
    if (token < end) entry = p.table[(int64_t)r.request * p.ld_table + column];  // (end is inside the table)
    const bool ok = entry >= 0 && entry < p.cache.pages;
    there = __ballot(ok);
    const int64_t begins = (ok ? entry : 0) * p.cache.page_bytes, within = token - column * page;
    codes_at = begins + within * (D / 2), pairs_at = begins + within * 4;
  };
  auto from_lane = [&](int64_t v, int l) __attribute__((always_inline)) {
    return (int64_t)((uint64_t)(u32)__builtin_amdgcn_readlane((int)((uint64_t)v >> 32), l) << 32 | (u32)__builtin_amdgcn_readlane((int)v, l));
  };
  // A block's keys, values and pairs.  Those of the next one are asked for as soon as the registers of this one's are free: values and pairs once they are in
  // LDS, keys behind their products.
  Dwords<W> keys[4], values[4];
  u32 key_pair, value_pair;
  const char *tiles[4];  // where they begin
  auto find = [&](int n) __attribute__((always_inline)) {
    if (n % 16 == 0) look_up(n);
    for (int j = 0; j < 4; j++) tiles[j] = cache + from_lane(codes_at, n % 16 * 4 + j);
  };
  u32 mine_at = m * (D / 2) + g * (4 * W);
  // (kept in 32 bits where it is used: a load takes a scalar address and an offset of that size)
  auto from_tile = [&](const char *tile) __attribute__((always_inline)) {
    asm("" : "+v"(mine_at));
    return load_dwords<W>(tile + mine_at);
  };
  auto load_keys = [&]() __attribute__((always_inline)) {
    for (int j = 0; j < 4; j++) keys[j] = from_tile(tiles[j]);
  };
  auto load_values = [&](int n) __attribute__((always_inline)) {
    for (int j = 0; j < 4; j++) values[j] = from_tile(tiles[j] + (int64_t)page * (D / 2));
    const int at = n % 16 * 4 + g, token = start + n * STEP + lane;
    const char *pairs = cache + (int64_t)page * D + __shfl(pairs_at, at) + m * 4;
    key_pair = *(const u32 *)pairs, value_pair = *(const u32 *)(pairs + page * 4);
    if (token >= end || !(there >> at & 1)) key_pair = value_pair = 0;  // (memory that was never written may hold any)
  };

  if (blocks) {
    find(0);
    load_values(0);
    load_keys();
  }
  // q as operands
  // (A score in powers of two is factor * lift * (codes' product * step + lowest * sum of q): the lift is 1, but 2^40 where 32 bits cannot hold the factor without it, of rows with elements of 2^85 and
  // more.  It holds wherever the scale times the row's largest element is finite in 32 bits.)
  float factor[RT], sum_q[RT];
  uint4 q[RT][W];
  bool lifted = false;
  for (int t = 0; t < RT; t++) {
    float v[W][8], most = 0.f, sum = 0.f;
    for (int w = 0; w < W; w++)
      for (int e = 0; e < 8; e++) {
        v[w][e] = half_of(raw[t][w].d[e / 2], BF16, e & 1);  // (of a row that is not there: the first's, for nothing)
        most = fmaxf(most, fabsf(v[w][e]));
      }
    most = over_row(most, [](float a, float b) { return fmaxf(a, b); });
    const int power_q = most > 0.f && most < __builtin_inff() ? max(-126, min(126, 14 - __builtin_amdgcn_frexp_expf(most))) : 0;
    const float sign = __builtin_amdgcn_ldexpf(p.scale < 0.f ? -1.f : p.scale == 0.f ? 0.f : 1.f, power_q);
    for (int w = 0; w < W; w++) {
      float x[8];
      for (int e = 0; e < 8; e++) x[e] = v[w][e] * (e & 2 ? sign * 0x1p-4f : sign), sum += v[w][e] * sign;
      q[t][w] = make_uint4(fp16_pair(x[0], x[1]), fp16_pair(x[2], x[3]), fp16_pair(x[4], x[5]), fp16_pair(x[6], x[7]));
    }
    sum = over_row(sum, [](float a, float b) { return a + b; });
    const bool far = !(__builtin_amdgcn_ldexpf(fabsf(p.scale), 24 - power_q) < 0x1p100f);
    factor[t] = fmaxf(__builtin_amdgcn_ldexpf(fabsf(p.scale), (far ? -16 : 24) - power_q) * LOG2_E, 0x1p-149f);
    // (a row with an infinity: NaN, as the formula gives, also where all its scores are -inf here)
    sum_q[t] = (sum - sum == 0.f ? sum : __builtin_nanf("")) * (far ? 0x1p16f : 0x1p-24f);
    lifts[t * ROWS + m % ROWS] = far ? 0x1p40f : 1.f, powers[t * ROWS + m % ROWS] = -112;
    lifted = lifted || __any(far);
  }
  f32x4 out[D / 16][RT];
  float top[RT], total[RT], lowest[RT];
  for (int t = 0; t < RT; t++) {
    top[t] = -__builtin_inff(), total[t] = 0.f, lowest[t] = 0.f;
    for (int d = 0; d < D / 16; d++) out[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The rows' powers are the same as a rule, and value_step holds steps in their unit.  Where they are not (some have seen a larger step than others), or where rows must not see one that is past their
  // power, it holds steps as they are, for each row to take in its own unit.
  bool mixed = false;
  float unit = 0x1p126f, limit = 0x1p-112f;  // of the least power; 2^ it
  bool far[RT] = {};                         // exponents of some row are of the difference to its maximum

  for (int n = 0; n < blocks; n++) {
    const u32 present = (u32)(there >> (n % 16 * 4)) & 15;  // tiles
    // values and pairs to LDS: the 16 tokens of a lane's operand in a row, 8 bytes between rows
    for (int j = 0; j < 4; j++) __builtin_memcpy(mine + (m / 4 * 16 + j * 4 + m % 4) * PITCH + g * (4 * W), &values[j], 4 * W);
    const float step = half_of(value_pair, BF16, false), lowest_value = half_of(value_pair, BF16, true);
    const int first = start + n * STEP;
    const bool whole = first >= seen_from && first + BLOCK <= seen_to && present == 15;
    const bool raises = step >= limit && step < __builtin_inff();
    if (__builtin_expect(__any(raises), 0)) {  // the largest so far, for some row: what there is in its unit
      const bool here = present >> g & 1, by_all = here && first + lane >= seen_from && first + lane < seen_to;
      const float largest = over_lanes<64>(raises && by_all ? step : 0.f, [](float a, float b) { return fmaxf(a, b); });
      const float reach = largest > 0.f ? __builtin_amdgcn_ldexpf(1.f, __builtin_amdgcn_frexp_expf(largest)) : 0.f;
      float most[RT];
      for (int t = 0; t < RT; t++) most[t] = largest;
      if (__any(raises && !by_all && step >= reach)) {  // (of the others none matters beside what all rows see)
        value_step[lane] = raises && here ? step : 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int t = 0; t < RT; t++) {
          const int from = low[t] - first - 16 * g, to = min(high[t], end) - first - 16 * g;
          float seen = 0.f;
          for (int i = 0; i < 16; i += 4) {
            const f32x4 steps = *(const f32x4 *)(value_step + 16 * g + i);
            for (int e = 0; e < 4; e++) seen = fmaxf(seen, i + e >= from && i + e < to ? steps[e] : 0.f);
          }
          most[t] = over_row(seen, [](float a, float b) { return fmaxf(a, b); });
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      int least = 1024, greatest = -1024;
      for (int t = 0; t < RT; t++) {
        const int was = powers[t * ROWS + m % ROWS], now = most[t] > 0.f ? max(was, __builtin_amdgcn_frexp_expf(most[t])) : was;
        const float moved = __builtin_amdgcn_ldexpf(1.f, max(was - now, -126));
        for (int d = 0; d < D / 16; d++)
          for (int i = 0; i < 4; i++) out[d][t][i] *= moved;
        powers[t * ROWS + m % ROWS] = now;
        if (high[t] > 0) least = min(least, now), greatest = max(greatest, now);  // (not of rows that are not there)
      }
      least = over_lanes<16>(least, [](int a, int b) { return min(a, b); }), greatest = over_lanes<16>(greatest, [](int a, int b) { return max(a, b); });
      least = __builtin_amdgcn_readfirstlane(least), mixed = __builtin_amdgcn_readfirstlane(greatest) != least;
      unit = __builtin_amdgcn_ldexpf(1.f, 14 - least), limit = __builtin_amdgcn_ldexpf(1.f, least);
    }
    // a step or lowest value of NaN stays with the rows that see it: 0 times it is not 0
    const bool careful = mixed || (!whole && __any(!(fabsf(step) + fabsf(lowest_value) < __builtin_inff()) || step >= limit));
    const float steps_unit = careful ? 1.f : unit;
    key_step[lane] = half_of(key_pair, BF16, false), key_low[lane] = half_of(key_pair, BF16, true);
    value_step[lane] = step * (lane & 1 ? steps_unit * 0x1p-4f : steps_unit), value_low[lane] = lowest_value;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (n + 1 < blocks) {
      find(n + 1);
      load_values(n + 1);
    }

    f32x4 s[NJ][RT];  // of tiles NJ * bank ..
    {
      f32x4 all[4][RT];
      for (int j = 0; j < 4; j++) {
        for (int t = 0; t < RT; t++) all[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < W; w++) {
          const uint4 k = codes_of(keys[j].d[w]);
          for (int t = 0; t < RT; t++) all[j][t] = mfma16<false>(k, q[t][w], all[j][t]);
        }
      }
      for (int t = 0; t < RT; t++)
        for (int j = 0; j < NJ; j++)
          for (int i = 0; i < 4; i++) {
            s[j][t][i] = all[j][t][i];
            for (int b = 1; b < BANKS; b++) s[j][t][i] = bank == b ? all[NJ * b + j][t][i] : s[j][t][i];
          }
    }
    if (n + 1 < blocks) load_keys();
    if (__builtin_expect(lifted, 0))
      for (int t = 0; t < RT; t++) {
        const float lift = lifts[t * ROWS + m % ROWS];
        for (int j = 0; j < NJ; j++)
          for (int i = 0; i < 4; i++) s[j][t][i] *= lift;
      }
    const int at = 16 * NJ * bank + 4 * g;  // the first of a lane's tokens in the block
    for (int j = 0; j < NJ; j++) {
      const f32x4 step_k = *(const f32x4 *)(key_step + at + 16 * j), low_k = *(const f32x4 *)(key_low + at + 16 * j);
      for (int t = 0; t < RT; t++)
        for (int i = 0; i < 4; i++) s[j][t][i] = __builtin_fmaf(s[j][t][i], step_k[i], low_k[i] * sum_q[t]);
    }
    if (!whole)
      for (int t = 0; t < RT; t++) {
        const int from = low[t] - first - at, to = min(high[t], end) - first - at;
        for (int j = 0; j < NJ; j++)
          for (int i = 0; i < 4; i++) s[j][t][i] = 16 * j + i >= from && 16 * j + i < to && (present >> (NJ * bank + j) & 1) ? s[j][t][i] : -__builtin_inff();
      }
    uint4 weights[RT][BF16 ? 1 : 2][2];
    for (int t = 0; t < RT; t++) {
      float most = -__builtin_inff();
      for (int j = 0; j < NJ; j++)
        for (int i = 0; i < 4; i++) most = fmaxf(most, s[j][t][i]);
      most = fmaxf(top[t], over_row<ROWS>(most, [](float a, float b) { return fmaxf(a, b); }));
      const float from = most == -__builtin_inff() ? 0.f : most, shift = -from * factor[t];  // (-inf: nothing seen yet)
      if (__any(most != top[t])) {
        const float kept = __builtin_amdgcn_exp2f((top[t] - from) * factor[t]);
        total[t] *= kept, lowest[t] *= kept;
        for (int d = 0; d < D / 16; d++)
          for (int i = 0; i < 4; i++) out[d][t][i] *= kept;
        top[t] = most;
        // (one rounding of the maximum instead of a difference per score: of up to 2^12 it is off by 2^-12, of 2^27 it would make weights of 16, or of 0)
        far[t] = __any(!(fabsf(shift) <= 0x1p12f));
      }
      float sum = 0.f, base = 0.f;
      auto weigh = [&](auto checked) __attribute__((always_inline)) {
        constexpr int J = NJ < 2 ? 1 : 2;  // tiles of a pair that are the lane's own
        constexpr bool apart = decltype(checked)::value;
        const bool by_difference = !(fabsf(shift) <= 0x1p12f);
        const float own = apart && careful ? __builtin_amdgcn_ldexpf(1.f, 14 - powers[t * ROWS + m % ROWS]) : 1.f;
        // pairs of tiles 0 and 1, and of 2 and 3, into the lanes of bank 0 (the others' columns of `out` hold nothing of use)
        for (int h = 0; h < NJ / J; h++) {
          float e[2][4], st[2][4];
          for (int j = 0; j < J; j++) {
            const f32x4 step_v = *(const f32x4 *)(value_step + at + 16 * (2 * h + j)), low_v = *(const f32x4 *)(value_low + at + 16 * (2 * h + j));
            for (int i = 0; i < 4; i++) {
              const float score = s[2 * h + j][t][i];
              const bool ok = !apart || score != -__builtin_inff();
              e[j][i] = __builtin_amdgcn_exp2f(apart && by_difference ? (score - from) * factor[t] : __builtin_fmaf(score, factor[t], shift));
              st[j][i] = !apart ? step_v[i] : ok ? step_v[i] * own : 0.f;
              sum += e[j][i];
              base = __builtin_fmaf(e[j][i], ok ? low_v[i] : 0.f, base);
            }
          }
          u32 w[4], rest[4];
          for (int i = 0; i < 4; i++) {
            const float a = e[0][i] * st[0][i], b = J == 1 ? dpp_moved<0x104>(a) : e[J - 1][i] * st[J - 1][i];  // (row_shl 4)
            w[i] = fp16_pair(a, b);
            if constexpr (!BF16) {
              // (of the operand's own halves: made a second time, from the product without its rounding, they may be the next ones)
              asm("" : "+v"(w[i]));
              const tts_gemm_device::f16x2 pair = __builtin_bit_cast(tts_gemm_device::f16x2, w[i]);
              const float ra = __builtin_fmaf(e[0][i], st[0][i], -(float)pair[0]);
              rest[i] = fp16_pair(ra, J == 1 ? dpp_moved<0x104>(ra) : __builtin_fmaf(e[J - 1][i], st[J - 1][i], -(float)pair[1]));
            }
          }
          weights[t][0][h] = make_uint4(w[0], w[1], w[2], w[3]);
          if constexpr (!BF16) weights[t][1][h] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        }
        if constexpr (NJ < 4)
          for (int part = 0; part < (BF16 ? 1 : 2); part++) {
            const uint4 w = weights[t][part][0];
            weights[t][part][1] = make_uint4(dpp_moved<0x108>(w.x), dpp_moved<0x108>(w.y), dpp_moved<0x108>(w.z), dpp_moved<0x108>(w.w));  // row_shl 8
          }
      };
      if (__builtin_expect(careful || far[t], 0)) weigh(std::true_type{});
      else weigh(std::false_type{});
      total[t] += sum, lowest[t] += base;
    }
    for (int d = 0; d < D / 16; d++) {
      const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32((i32x2 __attribute__((address_space(3))) *)((__attribute__((address_space(3))) void *)(mine + lane * PITCH + 8 * d)));
      for (int h = 0; h < 2; h++) {
        const uint4 c = codes_of(v[h]);
        for (int part = 0; part < (BF16 ? 1 : 2); part++)
          for (int t = 0; t < RT; t++) out[d][t] = mfma16<false>(c, weights[t][part][h], out[d][t]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  for (int t = 0; t < RT; t++) {
    const auto add = [](float a, float b) { return a + b; };
    total[t] = over_row<ROWS>(total[t], add), lowest[t] = over_row<ROWS>(lowest[t], add), top[t] *= factor[t];
    const int power = powers[t * ROWS + m % ROWS];
    for (int d = 0; d < D / 16; d++)
      for (int i = 0; i < 4; i++) out[d][t][i] = __builtin_amdgcn_ldexpf(out[d][t][i], 10 + power) + lowest[t];
  }
  // four elements of a row of the tile
  const int tile0 = r.tile * TILE, part0 = r.index + r.tile * r.slices + r.slice;
  auto put = [&](int row, int element, f32x4 v, float most, float sum) __attribute__((always_inline)) {
    const int token = divided(tile0 + row, p.by_group), head = kv * p.group + tile0 + row - token * p.group;
    if (token >= r.rows) return;
    if (r.slices == 1) {
      const float over = sum == 0.f ? 0.f : 1.f / sum;  // (a row that sees nothing: zeros)
      u32 w[2];
      for (int i = 0; i < 2; i++) {
        const float a = v[2 * i] * over, c = v[2 * i + 1] * over;
        w[i] = BF16 ? (u32)__builtin_bit_cast(uint16_t, (__bf16)a) | (u32)__builtin_bit_cast(uint16_t, (__bf16)c) << 16 : fp16_pair(a, c);
      }
      __builtin_memcpy((char *)p.out + 2 * ((int64_t)(r.first + token) * p.o_token + head * p.o_head + element), w, 8);
    } else {
      const int64_t part = ((int64_t)part0 * kv_heads + kv) * TILE + row;
      *(f32x4 *)(p.parts + part * D + element) = v;
      if (element == 0) p.stats[part * 2] = most, p.stats[part * 2 + 1] = sum;
    }
  };
  if constexpr (OWN != OWN_BLOCKS) {
    if (bank == 0)
      for (int t = 0; t < RT; t++)
        for (int d = 0; d < D / 16; d++) put(row0 - tile0 + t * ROWS + m, 16 * d + 4 * g, out[d][t], top[t], total[t]);
  } else {  // the wavefronts' parts meet in LDS
    float *const rows = (float *)lds, *const tops = rows + WAVES * WAVE_ROWS * MEET_PITCH, *const totals = tops + WAVES * WAVE_ROWS;
    __syncthreads();
    if (bank == 0)
      for (int t = 0; t < RT; t++) {
        const int row = wave * WAVE_ROWS + t * ROWS + m;
        for (int d = 0; d < D / 16; d++) *(f32x4 *)(rows + row * MEET_PITCH + 16 * d + 4 * g) = out[d][t];
        if (g == 0) tops[row] = top[t], totals[row] = total[t];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < WAVE_ROWS * (D / 4); i += 256) {
      const int row = i / (D / 4), element = i % (D / 4) * 4;
      float most = tops[row], sum = 0.f;
      for (int w = 1; w < WAVES; w++) most = fmaxf(most, tops[w * WAVE_ROWS + row]);
      const float base = most == -__builtin_inff() ? 0.f : most;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < WAVES; w++) {
        const float share = __builtin_amdgcn_exp2f(tops[w * WAVE_ROWS + row] - base);
        sum += totals[w * WAVE_ROWS + row] * share;
        const f32x4 part = *(const f32x4 *)(rows + (w * WAVE_ROWS + row) * MEET_PITCH + element);
        for (int e = 0; e < 4; e++) v[e] += part[e] * share;
      }
      put(row, element, v, most, sum);
    }
  }
}

// The slices of a row, where there are several, added up in their order by TPR threads: four elements a thread, and as many slices side by side as that leaves.
template <bool BF16, int TPR>
__global__ __launch_bounds__(256) void kv4_attend_join_kernel(AttendParams p) {
  __shared__ float shares_of[256 / TPR][MOST_SLICES];
  __shared__ f32x4 sums[256];
  const int tid = threadIdx.x % TPR, lane = threadIdx.x % 64, dim = p.cache.dim, row = blockIdx.x * (256 / TPR) + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const int token = divided(row, p.by_heads), head = row - token * p.heads;
  if (token >= p.tokens) return;
  const Work r = work_of(p, -1, token);
  if (!r.rows || r.slices == 1) return;  // a row of no request, or written already
  const int kv = divided(head, p.by_group), in_request = (token - r.first) * p.group + head - kv * p.group, tile = 1 << p.plan.tile_log;
  const int64_t part_step = (int64_t)p.cache.heads * tile;  // from slice to slice
  const int64_t index = r.index + (int64_t)(in_request >> p.plan.tile_log) * r.slices;
  if (index + r.slices > p.plan.items + p.plan.extra) return;  // (only where starts are not in order)
  const int64_t first = (index * p.cache.heads + kv) * tile + (in_request & (tile - 1));
  const float *stats = p.stats + first * 2, *parts = p.parts + first * dim;
  const int four = dim <= 32 ? 8 : dim <= 64 ? 16 : dim <= 128 ? 32 : 64, at = tid % four, side = TPR / four;  // threads per slice, their element, slices at a time
  const bool mine = 4 * at < dim;
  // (the first four of a thread's on their way together, and the statistics with them)
  f32x4 part[4];
  for (int n = 0; n < 4; n++)
    if (mine && tid / four + n * side < r.slices) part[n] = *(const f32x4 *)(parts + (tid / four + n * side) * part_step * dim + 4 * at);
  // (every wavefront for itself)
  float top[2], total[2], most = -__builtin_inff(), all = 0.f;
  for (int h = 0; h < 2; h++) {
    const int i = lane + 64 * h;
    top[h] = i < r.slices ? stats[2 * i * part_step] : -__builtin_inff(), total[h] = i < r.slices ? stats[2 * i * part_step + 1] : 0.f;
    most = fmaxf(most, top[h]);
  }
  most = over_lanes<64>(most, [](float a, float b) { return fmaxf(a, b); });
  const float base = most == -__builtin_inff() ? 0.f : most;
  float *shares = shares_of[threadIdx.x / TPR];
  for (int h = 0; h < 2; h++) {
    const float share = __builtin_amdgcn_exp2f(top[h] - base);
    all += total[h] * share;
    if (tid < 64) shares[lane + 64 * h] = share;
  }
  all = over_lanes<64>(all, [](float a, float b) { return a + b; });
  auto meet = [&]() __attribute__((always_inline)) {
    if constexpr (TPR > 64) __syncthreads();
    else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  meet();
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int n = 0; n < 4; n++)
    if (mine && tid / four + n * side < r.slices)
      for (int e = 0; e < 4; e++) sum[e] += part[n][e] * shares[tid / four + n * side];
  for (int i = tid / four + 4 * side; mine && i < r.slices; i += side) {
    const f32x4 next = *(const f32x4 *)(parts + i * part_step * dim + 4 * at);
    for (int e = 0; e < 4; e++) sum[e] += next[e] * shares[i];
  }
  sums[threadIdx.x] = sum;
  meet();
  if (tid >= four || !mine) return;
  for (int i = 1; i < min(side, r.slices); i++)
    for (int e = 0; e < 4; e++) sum[e] += sums[threadIdx.x + i * four][e];
  const float over = all == 0.f ? 0.f : 1.f / all;
  uint16_t out[4];
  for (int e = 0; e < 4; e++) out[e] = BF16 ? __builtin_bit_cast(uint16_t, (__bf16)(sum[e] * over)) : __builtin_bit_cast(uint16_t, (_Float16)(sum[e] * over));
  __builtin_memcpy((uint16_t *)p.out + (int64_t)token * p.o_token + head * p.o_head + 4 * at, out, sizeof out);
}

template <bool BF16, int W>
hipError_t launch_of(const AttendParams &p, hipStream_t s) {
  const int per_item = p.plan.own == OWN_HEADS ? (p.cache.heads + WAVES - 1) / WAVES : p.cache.heads;
  AttendParams q = p;
  q.by_per_item = fast_div(per_item);
  const dim3 grid((unsigned)((p.plan.items + p.plan.extra) * per_item + (p.clear ? 8 : 0)));
  auto go = [&](auto rows) __attribute__((always_inline)) {
    constexpr int ROWS = decltype(rows)::value;
    if (p.plan.own == OWN_HEADS) kv4_attend_kernel<BF16, W, 1, ROWS, OWN_HEADS><<<grid, 256, 0, s>>>(q);
    else kv4_attend_kernel<BF16, W, 1, ROWS, OWN_BLOCKS><<<grid, 256, 0, s>>>(q);
  };
  if (p.plan.own == OWN_ROWS) kv4_attend_kernel<BF16, W, row_tiles_of(W), 16, OWN_ROWS><<<grid, 256, 0, s>>>(q);
  else if (p.plan.tile_log == 2) go(row_ops::Int<4>{});
  else if (p.plan.tile_log == 3) go(row_ops::Int<8>{});
  else go(row_ops::Int<16>{});
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.plan.extra) {
    const unsigned rows = (unsigned)(p.tokens * p.heads);
    // (64 ragged requests of 32 heads 34.5 us in all, with 256 threads a row 35.9; 2 requests of 64 heads 42.6 and 37.0)
    if (rows >= 1024) kv4_attend_join_kernel<BF16, 64><<<dim3((rows + 3) / 4), 256, 0, s>>>(p);
    else kv4_attend_join_kernel<BF16, 256><<<dim3(rows), 256, 0, s>>>(p);
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

// Which kernel, and how many workgroups.  Both sides of each rule as measured, us a call in a graph, dim 128 and 8 heads of the cache where nothing else is said:
// * Rows of their own for each wavefront where a request has 128 and more on average and they make 384 workgroups: 64 requests of 256 rows 394 (shared blocks 466), 16 of 512 209
//   (220), but 16 of 256 158 (120) and 4 of 1024 132 (95): fewer workgroups do not fill the device, and the tokens are what is left to divide.
// * Heads of their own for each wavefront where there are 4 requests and heads for each token of the longest: 256 requests of 250 17.2 (shared blocks 27.1), 128 of up to 60 7.7 (12.8), 512 of up to 60
//   21.4 (42.5), 512 of up to 1000 44.5 (59.8), but 64 of up to 250 10.7 (8.4), 128 of up to 1000 26.3 (19.2); between them 256 of up to 1000 28.8 (30.3, and by the rule shared): what a workgroup does before and after
//   its blocks counts for four heads, and a head's blocks come one after another.
// * Tiles of 4 or 8 rows where a request has no more: 16 requests of 4000 tokens, 4 rows 21.3 (tiles of 8 21.6, of 16 22.6), 8 rows 21.4 (of 16 22.9, of 4 29.2).
// * Slices, of 512 workgroups beyond the tiles', where the longest request has more than 1024 tokens and 6 for each tile: 64 requests of up to 8192 35.2 (none: 47.5),
//   128 of up to 8000 65 (72), one of 1500 11.8 (12.8), but 128 of 4000 112 (109), 256 of up to 2000 53.0 (39.0), one of 600 11.6 (9.2): the second kernel, and what a
//   workgroup does before its first block and behind its last.
// All of them are batches of one number of new tokens for every request, and the average is all that the rules know: of others they may choose badly.  2048 rows of a prompt take 86 alone and 7 tokens of up
// to 8192 19, in one call 252 (of up to 131072 136, in one call 3771: a wavefront with rows of its own walks all of their tokens); 64 single tokens 65, padded to 8192 rows 590.
AttendPlan plan_attend(int64_t tokens, int requests, int heads, int kv_heads, int dim, int64_t longest, int window) {
  AttendPlan plan = {};
  const int64_t group = heads / kv_heads, rows = (tokens + requests - 1) / std::max(requests, 1) * group;  // of a request, on average
  const int64_t wide = WAVES * 16 * row_tiles_of(dim / 32);
  // tiles: each request's rows rounded up, which is what they are where a token's rows fill whole tiles
  auto tiles = [&](int64_t tile) { return std::max<int64_t>(1, group % tile == 0 ? tokens * (group / tile) : (tokens * group + requests * (tile - 1)) / tile); };
  const bool by_rows = rows >= 128 && tiles(wide) * kv_heads >= 384;
  const int64_t tile = by_rows ? wide : rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  plan.tile_log = __builtin_ctzll(tile);
  plan.items = tiles(tile);
  const int64_t range = window ? std::min<int64_t>(longest, (int64_t)window + tile / group + 17) : longest;
  plan.own = by_rows ? OWN_ROWS : kv_heads >= WAVES && 4 * range <= plan.items * kv_heads ? OWN_HEADS : OWN_BLOCKS;
  if (plan.own == OWN_BLOCKS && range > 1024 && 6 * plan.items * kv_heads <= range && tokens * heads < (1 << 24)) {  // (as many workgroups join them, and a launch has less than 2^32 lanes)
    const int64_t most = plan.items * std::min<int64_t>((range + BLOCK - 1) / BLOCK / WAVES, MOST_SLICES);  // (more than that has nothing to do)
    plan.extra = std::min((512 + kv_heads - 1) / (int64_t)kv_heads, most);
    plan.over_extra = 1.f / (float)plan.extra;
  }
  return plan;
}

size_t attend_workspace_bytes(const AttendPlan &plan, int kv_heads, int dim) {
  return plan.extra ? (size_t)(plan.items + plan.extra) * (kv_heads * (dim + 2) * sizeof(float) << plan.tile_log) : 0;
}

hipError_t launch_attend(const AttendParams &p, hipStream_t s) { return p.cache.bf16 ? launch_as<true>(p, s) : launch_as<false>(p, s); }

}  // namespace tts
