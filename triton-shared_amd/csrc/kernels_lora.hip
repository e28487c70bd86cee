// Low-rank adapters of many requests, added to what a shared projection made: with d = ids[t],
//   out[t] = base[t] + scales[d] * (x[t] A[d]^T) B[d]^T,    A[d]: rank x inputs, B[d]: outputs x rank;   out[t] = base[t] where d names none.
// Kernel 1 makes v = x A^T, kernel 2 adds scales * v B^T.  Both take tiles of neighbouring rows and go through the adapters that occur
// among a tile's rows, one product of all of them with each adapter, of which its own rows are kept: an adapter is read once per tile.
// In a prompt a tile has one adapter, in a decode batch up to one per row.  (The other rows are left out of the sums, not
// multiplied by zero: an infinity in one request's adapter stays with that request.)
// v is summed and kept in 32 bits, in slices of the inputs that kernel 2 adds as it reads them; it enters the second product as
// two 16-bit parts (row_device.h).
// What has to move is x, base and out once and the adapters.  What bounds it: few rows, the launches and chains of loads (one row of 4096 x 4096, rank
// 16: 4 + 7 us; 64 rows with an adapter each, 4096 x 8192: 10 + 15 us, up to 16 adapters in turn per tile, eight loads ahead); prompts of 8192 rows, rank 64:
// kernel 1 is one round of one workgroup per CU (64 rows take the registers of a SIMD for one wavefront), whose first loads and last sums nothing
// overlaps, 37 us for 67 MB of x; kernel 2, two workgroups per CU, reads B for every 32 rows, 134 MB from L2 beside as much of base and out, 60 us.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

using namespace row_ops;

constexpr int MAX_SLICES = 16;

struct Shape {
  int row_tiles, row_tiles_of_2, slices;  // (of kernel 1, of kernel 2)
  int columns_each;  // tiles of 256 columns that a workgroup of kernel 2 does one after another
  int64_t pitch_v;  // floats between rows of v: the rank, up to a multiple of 8
  size_t bytes;
};

// The adapters of a tile of up to 64 rows: lane i of a wavefront holds the i'th, in order of first occurrence; returns their number.
// `id`: the lane's row's, negative for none.
__device__ __forceinline__ int adapters_of(int id, int &mine) {
  const int lane = threadIdx.x & 63;
  uint64_t left = __ballot(id >= 0);
  int n = 0;
  mine = -1;
  while (left) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    left &= ~__ballot(id == cur);
    if (lane == n) mine = cur;
    n++;
  }
  return n;
}

__device__ __forceinline__ int row_id(const LoraParams &p, int64_t row) {
  if (row >= p.tokens) return -1;
  const int id = p.ids[row * p.stride_ids];
  return (u32)id < (u32)p.adapters ? id : -1;
}

// eight 16-bit elements from any element's address
__device__ __forceinline__ uint4 octet(const char *p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// ... the first `valid` of them, zeros behind, by how rows end.  (The checks at every load would be most of a kernel's code, and a launch for few rows waits for its code.)
enum Ends { EXACT = 3,  // with a whole step of 64
            EVEN = 0,   // with a whole octet
            LONG = 1,   // anywhere, at least eight elements from their beginning: the last octet's load is moved back to end with the row
            SHORT = 2 };
template <int ENDS>
__device__ __forceinline__ uint4 octet_part(const char *p, int valid) {
  if constexpr (ENDS == EXACT) return octet(p);
  else if constexpr (ENDS == EVEN) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (valid > 0) v = octet(p);
    return v;
  } else if constexpr (ENDS == LONG)
    return __builtin_bit_cast(uint4, load_part(p, 2 * valid));
  if (valid >= 8) return octet(p);
  u32 w[4] = {0, 0, 0, 0};
  for (int i = 0; i < valid; i++) w[i >> 1] |= (u32)((const uint16_t *)p)[i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- kernel 1: v[slice][t][r], 16 * MT rows and 16 * NB of the rank per workgroup; four wavefronts share the slice's steps of 64
// inputs, of which a row's 128 bytes are loaded at once.
// A tile with one adapter runs its steps in a ring of loads; one with several goes through steps and adapters in one sequence, the adapter
// changing fastest, and keeps of each product the rows that it belongs to.
template <bool BF16, int ENDS, int MT, int NB>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p, Shape sh, float *v) {
  constexpr int PITCH = 16 * NB + 4;
  __shared__ float red[4 * 16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (16 * MT);
  const int r0 = blockIdx.z * (16 * NB);
  const int my_id = lane < 16 * MT ? row_id(p, row0 + lane) : -1;
  const int K = (int)p.inputs, steps = (K + 63) / 64;
  const int share = (int)blockIdx.y * 4 + wave, shares = sh.slices * 4;
  const int begin = (int)((int64_t)share * steps / shares), end = (int)((int64_t)(share + 1) * steps / shares);
  const char *x[MT];
  each<0, MT>([&](auto mc) __attribute__((always_inline)) {
    const int64_t row = row0 + 16 * mc.value + c;
    x[mc.value] = (const char *)p.x + 2 * ((row < p.tokens ? row : p.tokens - 1) * p.ld_x + 8 * g);
  });
  u32 a_off[NB];
  each<0, NB>([&](auto ic) __attribute__((always_inline)) { a_off[ic.value] = (u32)(2 * (min(r0 + 16 * ic.value + c, p.rank - 1) * p.a_rank + 8 * g)); });
  int mine;
  const int n = adapters_of(my_id, mine);
  if (n == 0) return;  // (kernel 2 reads none of these rows)
  auto adapter = [&](int d) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(mine, d); };
  auto weights_of = [&](int cur) __attribute__((always_inline)) { return (const char *)p.a + 2 * ((int64_t)cur * p.a_adapter); };
  f32x4 acc[MT][NB];
  each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
  // (halves: k 8 g .. and 32 + 8 g ..)
  auto load_x = [&](int s, uint4 (&xs)[2][MT]) __attribute__((always_inline)) {
    each<0, 2 * MT>([&](auto nc) __attribute__((always_inline)) { xs[nc.value % 2][nc.value / 2] = octet_part<ENDS>(x[nc.value / 2] + 128 * (int64_t)s + 64 * (nc.value % 2), K - 64 * s - 32 * (nc.value % 2) - 8 * g); });
  };
  auto load_a = [&](const char *a, int s, uint4 (&as)[2][NB]) __attribute__((always_inline)) {
    const char *at = a + 128 * (int64_t)s;
    each<0, 2 * NB>([&](auto nc) __attribute__((always_inline)) { as[nc.value % 2][nc.value / 2] = octet_part<ENDS>(at + a_off[nc.value / 2] + 64 * (nc.value % 2), K - 64 * s - 32 * (nc.value % 2) - 8 * g); });
  };
  auto add = [&](const uint4 (&xs)[2][MT], const uint4 (&as)[2][NB]) __attribute__((always_inline)) {
    each<0, 2 * MT * NB>([&](auto nc) __attribute__((always_inline)) {
      constexpr int h = nc.value / (MT * NB), m = nc.value / NB % MT, i = nc.value % NB;
      acc[m][i] = mfma16<BF16>(xs[h][m], as[h][i], acc[m][i]);
    });
  };
  if (n == 1) {
    constexpr int U = MT + NB >= 4 ? 2 : 4;
    const char *a = weights_of(adapter(0));
    uint4 xs[U][2][MT], as[U][2][NB];
    if (begin < end) {
      each<0, U>([&](auto uc) __attribute__((always_inline)) {
        const int s = min(begin + uc.value, end - 1);
        load_x(s, xs[uc.value]);
        load_a(a, s, as[uc.value]);
      });
      int s = begin;
      for (; s + U <= end; s += U)
        each<0, U>([&](auto uc) __attribute__((always_inline)) {
          add(xs[uc.value], as[uc.value]);
          __builtin_amdgcn_sched_barrier(0);
          const int next = min(s + U + uc.value, end - 1);
          load_x(next, xs[uc.value]);
          load_a(a, next, as[uc.value]);
          __builtin_amdgcn_sched_barrier(0);
        });
      each<0, U>([&](auto uc) __attribute__((always_inline)) {
        if (s + uc.value < end) add(xs[uc.value], as[uc.value]);
      });
    }
  } else {
    int of_sum[MT][4];  // the adapters of the rows whose sums the lane holds
    each<0, MT * 4>([&](auto nc) __attribute__((always_inline)) { of_sum[nc.value / 4][nc.value % 4] = __shfl(my_id, 16 * (nc.value / 4) + 4 * g + nc.value % 4); });
    auto add_own = [&](const uint4 (&xs)[2][MT], const uint4 (&as)[2][NB], int cur) __attribute__((always_inline)) {
      each<0, MT * NB>([&](auto nc) __attribute__((always_inline)) {
        constexpr int m = nc.value / NB, i = nc.value % NB;
        const f32x4 sum = mfma16<BF16>(xs[1][m], as[1][i], mfma16<BF16>(xs[0][m], as[0][i], (f32x4){0.f, 0.f, 0.f, 0.f}));
        each<0, 4>([&](auto rc) __attribute__((always_inline)) { acc[m][i][rc.value] = of_sum[m][rc.value] == cur ? acc[m][i][rc.value] + sum[rc.value] : acc[m][i][rc.value]; });
      });
    };
    constexpr int U = NB >= 4 ? 2 : NB > 1 ? 4 : 8;
    uint4 xs[2][MT], xn[2][MT], as[U][2][NB];
    if (begin < end) {
      int fs = begin, fd = 0;  // what is fetched next
      auto fetch = [&](uint4 (&to)[2][NB]) __attribute__((always_inline)) {
        load_a(weights_of(adapter(fd)), fs, to);
        if (++fd == n) fd = 0, fs = min(fs + 1, end - 1);
      };
      load_x(begin, xs);
      load_x(min(begin + 1, end - 1), xn);
      each<0, U>([&](auto uc) __attribute__((always_inline)) { fetch(as[uc.value]); });
      int s = begin, d = 0;
      const int all = (end - begin) * n;
      for (int i = 0; i < all; i += U)
        each<0, U>([&](auto uc) __attribute__((always_inline)) {
          if (i + uc.value < all) {
            add_own(xs, as[uc.value], adapter(d));
            if (++d == n) {
              d = 0, s++;
              each<0, 2 * MT>([&](auto nc) __attribute__((always_inline)) { xs[nc.value % 2][nc.value / 2] = xn[nc.value % 2][nc.value / 2]; });
              load_x(min(s + 1, end - 1), xn);
            }
          }
          fetch(as[uc.value]);
        });
    }
  }
  each<0, MT>([&](auto mc) __attribute__((always_inline)) {
    constexpr int m = decltype(mc)::value;
    each<0, NB>([&](auto ic) __attribute__((always_inline)) {
      each<0, 4>([&](auto rc) __attribute__((always_inline)) { red[(wave * 16 + 4 * g + rc.value) * PITCH + 16 * ic.value + c] = acc[m][ic.value][rc.value]; });
    });
    __syncthreads();
    const int r = tid >> 4;
    const int64_t row = row0 + 16 * m + r;
    if (row < p.tokens)
      for (int j = tid & 15; j < 16 * NB && r0 + j < p.rank; j += 16) {
        float sum = 0.f;
        for (int q = 0; q < 4; q++) sum += red[(q * 16 + r) * PITCH + j];
        v[((int64_t)blockIdx.y * p.tokens + row) * sh.pitch_v + r0 + j] = sum;
      }
    __syncthreads();
  });
}

// ---- kernel 2: 16 * MT rows; a wavefront has 64 of every 256 columns.  The adapter goes in as the first operand: its row m (= lane % 16 of
// the load) of block i is column 16 (m / 4) + 4 i + m % 4, so that a lane's results are 16 neighbouring columns of row lane % 16.
// The rows' v comes through LDS, 128 of the rank at a time: slices added, scaled, in two parts.
template <bool BF16, int ENDS, int MT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p, Shape sh, const float *v) {
  constexpr int CHUNK = 128, PITCH = CHUNK + 8;
  __shared__ __align__(16) uint16_t parts[2][16 * MT][PITCH];
  __shared__ float row_back[16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
  const int my_id = lane < 16 * MT ? row_id(p, row0 + lane) : -1;
  int mine;
  const int n = adapters_of(my_id, mine);
  int id[MT];
  each<0, MT>([&](auto mc) __attribute__((always_inline)) { id[mc.value] = __shfl(my_id, 16 * mc.value + c); });
  // sixteen threads per row, eight values each
  auto stage = [&](int k0) __attribute__((always_inline)) {
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = 16 * mc.value + (tid >> 4), k = k0 + 8 * (tid & 15);
      const int of = __shfl(my_id, r);
      float f[8] = {};
      if (of >= 0 && k < p.rank) {
        const float *at = v + (row0 + r) * sh.pitch_v + k;
        const int64_t slice = p.tokens * sh.pitch_v;
        const float factor = p.scales ? p.scales[of] : 1.f;
        for (int q0 = 0; q0 < sh.slices; q0 += 8) {  // eight slices at a time on their way
          float4 a[8], b[8];
          each<0, 8>([&](auto qc) __attribute__((always_inline)) {
            const float *from = at + min(q0 + qc.value, sh.slices - 1) * slice;
            a[qc.value] = *(const float4 *)from, b[qc.value] = *(const float4 *)(from + 4);
          });
          each<0, 8>([&](auto qc) __attribute__((always_inline)) {
            if (q0 + qc.value < sh.slices) {
              const float4 s = a[qc.value], t = b[qc.value];
              f[0] += s.x, f[1] += s.y, f[2] += s.z, f[3] += s.w, f[4] += t.x, f[5] += t.y, f[6] += t.z, f[7] += t.w;
            }
          });
        }
        each<0, 8>([&](auto ic) __attribute__((always_inline)) { f[ic.value] = k + ic.value < p.rank ? f[ic.value] * factor : 0.f; });
      }
      float scale = 1.f;
      if constexpr (!BF16) {
        float most = 0.f;
        each<0, 8>([&](auto ic) __attribute__((always_inline)) { most = fmaxf(most, fabsf(f[ic.value])); });
        for (int d = 1; d < 16; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        scale = fp16_scale(most);
        if ((tid & 15) == 0) row_back[r] = 1.f / scale;
      }
      *(uint4 *)&parts[0][r][8 * (tid & 15)] = split_part<BF16, 0>(f, scale);
      *(uint4 *)&parts[1][r][8 * (tid & 15)] = split_part<BF16, 1>(f, scale);
    });
    __syncthreads();
  };
  // a tile's loads of base, and of the first adapters: on their way before v is staged, and before the tile before is stored
  constexpr int U = MT > 1 || ENDS != EVEN ? 2 : 4;
  const bool once = p.rank <= CHUNK;
  uint4 e[MT][2], ring[U][4];
  int64_t b_off[4], col = 0;
  int have = 0, fd = 0, fs = 0;
  auto fetch = [&](uint4 (&to)[4], int k0, int steps) __attribute__((always_inline)) {
    const char *b = (const char *)p.b + 2 * ((int64_t)__builtin_amdgcn_readlane(mine, fd) * p.b_adapter + k0 + 32 * fs);
    const int valid = p.rank - k0 - 32 * fs - 8 * g;
    each<0, 4>([&](auto ic) __attribute__((always_inline)) { to[ic.value] = octet_part<ENDS>(b + b_off[ic.value], valid); });
    if (++fs == steps) fs = 0, fd = min(fd + 1, n - 1);
  };
  auto begin = [&](int64_t tile, int k0) __attribute__((always_inline)) {
    fd = fs = 0;
    if (k0 == 0) {
      const int64_t col0 = tile * 256 + 64 * wave;
      col = col0 + 16 * g;
      have = (int)max((int64_t)0, min((int64_t)16, p.outputs - col));
      each<0, 4>([&](auto ic) __attribute__((always_inline)) {
        const int64_t from = col0 + 16 * (c >> 2) + 4 * ic.value + (c & 3);
        b_off[ic.value] = 2 * ((from < p.outputs ? from : p.outputs - 1) * p.b_col + 8 * g);
      });
    }
    const int steps = (min(CHUNK, p.rank - k0) + 31) / 32;
    if (n) each<0, U>([&](auto uc) __attribute__((always_inline)) { fetch(ring[uc.value], k0, steps); });
    if (k0 == 0)
      each<0, MT>([&](auto mc) __attribute__((always_inline)) {
        const int64_t row = row0 + 16 * mc.value + c;
        const char *base = (const char *)p.base + 2 * (row * p.ld_base + col);
        if (row < p.tokens) {
          if (have == 16) e[mc.value][0] = octet(base), e[mc.value][1] = octet(base + 16);
          else if (ENDS != EVEN) e[mc.value][0] = octet_part<ENDS>(base, have), e[mc.value][1] = octet_part<ENDS>(base + 16, have - 8);
        }
      });
  };
  const int64_t first = blockIdx.x * (int64_t)sh.columns_each, last = min(first + sh.columns_each, (p.outputs + 255) / 256);
  begin(first, 0);
  if (n && once) stage(0);
  for (int64_t tile = first; tile < last; tile++) {
    f32x4 acc[MT][4];
    each<0, MT * 4>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / 4][ic.value % 4] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
    for (int k0 = 0; n && k0 < p.rank; k0 += CHUNK) {
      if (!once) {
        stage(k0);
        if (k0) begin(tile, k0);
      }
      // adapters and steps of 32 of the rank in one sequence, U loads ahead
      const int steps = (min(CHUNK, p.rank - k0) + 31) / 32, all = n * steps;
      f32x4 sum[MT][4];
      each<0, MT * 4>([&](auto ic) __attribute__((always_inline)) { sum[ic.value / 4][ic.value % 4] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
      int d = 0, s = 0;
      for (int i = 0; i < all; i += U)
        each<0, U>([&](auto uc) __attribute__((always_inline)) {
          if (i + uc.value < all) {
            each<0, MT>([&](auto mc) __attribute__((always_inline)) {
              constexpr int m = decltype(mc)::value;
              const uint4 hi = *(const uint4 *)&parts[0][16 * m + c][32 * s + 8 * g], lo = *(const uint4 *)&parts[1][16 * m + c][32 * s + 8 * g];
              each<0, 4>([&](auto ic) __attribute__((always_inline)) { sum[m][ic.value] = mfma16<BF16>(ring[uc.value][ic.value], hi, sum[m][ic.value]); });
              each<0, 4>([&](auto ic) __attribute__((always_inline)) { sum[m][ic.value] = mfma16<BF16>(ring[uc.value][ic.value], lo, sum[m][ic.value]); });
            });
            if (++s == steps) {  // the adapter is done: its rows keep their sums
              const int cur = __builtin_amdgcn_readlane(mine, d);
              each<0, MT>([&](auto mc) __attribute__((always_inline)) {
                constexpr int m = decltype(mc)::value;
                const float back = BF16 ? 1.f : row_back[16 * m + c];
                each<0, 4>([&](auto ic) __attribute__((always_inline)) {
                  if (id[m] == cur) acc[m][ic.value] += sum[m][ic.value] * back;
                  sum[m][ic.value] = (f32x4){0.f, 0.f, 0.f, 0.f};
                });
              });
              s = 0, d++;
            }
          }
          if (i + uc.value + U < all) fetch(ring[uc.value], k0, steps);
        });
      if (!once) __syncthreads();
    }
    uint4 was[MT][2];
    each<0, 2 * MT>([&](auto nc) __attribute__((always_inline)) { was[nc.value / 2][nc.value % 2] = e[nc.value / 2][nc.value % 2]; });
    const int64_t col_now = col;
    const int have_now = have;
    if (tile + 1 < last) begin(tile + 1, 0);
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      const int64_t row = row0 + 16 * m + c;
      if (row >= p.tokens || have_now == 0) return;
      uint16_t now[16];
      __builtin_memcpy(now, was[m], 32);
      if (id[m] >= 0)  // (a row without an adapter is copied as it is)
        each<0, 16>([&](auto ic) __attribute__((always_inline)) {
          constexpr int i = decltype(ic)::value;
          const float old = BF16 ? __uint_as_float((u32)now[i] << 16) : (float)__builtin_bit_cast(_Float16, now[i]);
          const float made = old + acc[m][i / 4][i % 4];
          now[i] = BF16 ? tts_gemm_device::f32_to_bf16(made) : tts_gemm_device::f32_to_f16(made);
        });
      uint16_t *out = (uint16_t *)p.out + row * p.ld_out + col_now;
      if (have_now == 16) __builtin_memcpy(out, now, 32);
      else if (ENDS != EVEN) each<0, 16>([&](auto ic) __attribute__((always_inline)) { if (ic.value < have_now) out[ic.value] = now[ic.value]; });
    });
  }
}

constexpr int CUS = 256;

// Rows of a workgroup.  Few rows: as many workgroups as there can be.  Of prompts kernel 1 takes 64 (an adapter is read again for every
// tile: 8192 rows, rank 64: 36 us of 64, 43 of 32) and kernel 2 32 (it holds base and the sums: 59 us of 32, 82 of 64).  Both kernels of 4096 x 4096, us of
// 16 rows and of 64 / 32: rank 16, one adapter, 512 rows 12 and 15, 1024 rows 18 and 19, 2048 rows 25 and 24, 4096 rows 45 and 39; 64 adapters row by
// row 30 and 52, 47 and 58, 80 and 95, 148 and 170; rank 64, one adapter 18 and 21, 26 and 24, 40 and 32, 71 and 47; 64 adapters 71 and 103, 125 and 129,
// 239 and 229, 467 and 434.
bool many_rows(const LoraParams &p) { return p.tokens > 1024; }

Shape shape_of(const LoraParams &p) {
  Shape sh;
  const int64_t rows = many_rows(p) ? 64 : 16, rows_of_2 = many_rows(p) ? 32 : 16;
  sh.row_tiles = (int)std::max<int64_t>(1, (p.tokens + rows - 1) / rows);
  sh.row_tiles_of_2 = (int)std::max<int64_t>(1, (p.tokens + rows_of_2 - 1) / rows_of_2);
  // slices of the inputs until there is a workgroup per CU, of at least a step of 64 per wavefront
  const int steps = (int)((p.inputs + 63) / 64);
  sh.slices = std::max(1, std::min({MAX_SLICES, CUS / sh.row_tiles, steps / 4}));
  sh.pitch_v = (p.rank + 7) & ~7;
  // tiles of columns one after another, with v staged once, while that leaves two workgroups per CU (8192 rows of 4096: 59 us, 76 of a tile each)
  const int64_t column_tiles = (p.outputs + 255) / 256;
  sh.columns_each = (int)std::max<int64_t>(1, std::min<int64_t>(8, sh.row_tiles_of_2 * column_tiles / (2 * CUS)));
  sh.bytes = (size_t)sh.slices * p.tokens * sh.pitch_v * 4;
  return sh;
}

template <bool BF16, int MT1, int MT2>
hipError_t launch_rows(const LoraParams &p, const Shape &sh, hipStream_t s) {
  float *v = (float *)p.workspace;
  const int blocks = (p.rank + 15) / 16;
  auto shrink = [&](auto kernel, int nb) { kernel<<<dim3(sh.row_tiles, sh.slices, (blocks + nb - 1) / nb), 256, 0, s>>>(p, sh, v); };
  auto shrink_in = [&](auto ends) {
    constexpr int ENDS = decltype(ends)::value;
    if (blocks <= 1) shrink(lora_shrink_kernel<BF16, ENDS, MT1, 1>, 1);
    else if (blocks <= 2) shrink(lora_shrink_kernel<BF16, ENDS, MT1, 2>, 2);
    else shrink(lora_shrink_kernel<BF16, ENDS, MT1, 4>, 4);
  };
  auto expand_in = [&](auto ends) {
    lora_expand_kernel<BF16, decltype(ends)::value, MT2>
        <<<dim3((unsigned)(((p.outputs + 255) / 256 + sh.columns_each - 1) / sh.columns_each), sh.row_tiles_of_2), 256, 0, s>>>(p, sh, v);
  };
  if (p.inputs % 64 == 0) shrink_in(Int<EXACT>{});
  else if (p.inputs % 8 == 0) shrink_in(Int<EVEN>{});
  else if (p.inputs > 8) shrink_in(Int<LONG>{});
  else shrink_in(Int<SHORT>{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.rank % 8 == 0 && p.outputs % 16 == 0) expand_in(Int<EVEN>{});
  else if (p.rank >= 8 && p.outputs >= 8) expand_in(Int<LONG>{});
  else expand_in(Int<SHORT>{});
  return hipGetLastError();
}

}  // namespace

size_t lora_workspace_bytes(const LoraParams &p) { return shape_of(p).bytes; }

hipError_t launch_lora(const LoraParams &p, hipStream_t s) {
  const Shape sh = shape_of(p);
  if (many_rows(p)) return p.bf16 ? launch_rows<true, 4, 2>(p, sh, s) : launch_rows<false, 4, 2>(p, sh, s);
  return p.bf16 ? launch_rows<true, 1, 1>(p, sh, s) : launch_rows<false, 1, 1>(p, sh, s);
}

}  // namespace tts
