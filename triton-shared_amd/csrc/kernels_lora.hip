// Low-rank adapters of many requests, added to what a shared projection made: with d = ids[t],
//   out[t] = base[t] + scales[d] * (x[t] A[d]^T) B[d]^T,    A[d]: rank x inputs, B[d]: outputs x rank;   out[t] = base[t] where d names none.
// Kernel 1 makes v = x A^T, kernel 2 adds scales * v B^T.  Both take tiles of neighbouring rows and go through the adapters that occur
// among a tile's rows, one product of all of them with each adapter, of which its own rows are kept: an adapter is read once per tile.
// In a prompt a tile has one adapter, in a decode batch up to one per row.  (The other rows are left out of the sums, not
// multiplied by zero: an infinity in one request's adapter stays with that request.)
// v is summed and kept in 32 bits, in slices of the inputs that kernel 2 adds as it reads them; it enters the second product as
// two 16-bit parts (row_device.h).
// What has to move is x, base and out once and the adapters: memory or, for few rows, the launches.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

using namespace row_ops;

constexpr int MAX_SLICES = 32;

struct Shape {
  int row_tiles, slices;
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

// eight 16-bit elements from any element's address, the first `valid` of them; zero behind
__device__ __forceinline__ uint4 octet(const char *p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ uint4 octet_part(const char *p, int valid) {
  if (valid >= 8) return octet(p);
  u32 w[4] = {0, 0, 0, 0};
  for (int i = 0; i < valid; i++) w[i >> 1] |= (u32)((const uint16_t *)p)[i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- kernel 1: v[slice][t][r], 16 * MT rows and 16 * NB of the rank per workgroup; four wavefronts share the slice's steps of 32 inputs
template <bool BF16, int MT, int NB>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p, Shape sh, float *v) {
  constexpr int PITCH = 16 * NB + 4;
  __shared__ float red[4 * 16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (16 * MT);
  const int r0 = blockIdx.z * (16 * NB);
  int mine;
  const int n = adapters_of(lane < 16 * MT ? row_id(p, row0 + lane) : -1, mine);
  if (n == 0) return;  // (kernel 2 reads none of these rows)
  const char *x[MT];
  int of_sum[MT][4];  // the adapters of the rows whose sums the lane holds
  each<0, MT>([&](auto mc) __attribute__((always_inline)) {
    const int64_t row = row0 + 16 * mc.value + c;
    x[mc.value] = (const char *)p.x + 2 * ((row < p.tokens ? row : p.tokens - 1) * p.ld_x + 8 * g);
    each<0, 4>([&](auto rc) __attribute__((always_inline)) { of_sum[mc.value][rc.value] = row_id(p, row0 + 16 * mc.value + 4 * g + rc.value); });
  });
  int64_t a_off[NB];
  each<0, NB>([&](auto ic) __attribute__((always_inline)) { a_off[ic.value] = 2 * (min(r0 + 16 * ic.value + c, p.rank - 1) * p.a_rank + 8 * g); });
  const int K = (int)p.inputs, whole = K / 32, steps = (K + 31) / 32;
  const int share = (int)blockIdx.y * 4 + wave, shares = sh.slices * 4;
  const int begin = (int)((int64_t)share * steps / shares), end_all = (int)((int64_t)(share + 1) * steps / shares), end = min(end_all, whole);
  f32x4 acc[MT][NB];
  each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
  for (int d = 0; d < n; d++) {
    const int cur = __builtin_amdgcn_readlane(mine, d);
    const char *a = (const char *)p.a + 2 * ((int64_t)cur * p.a_adapter);
    f32x4 sum[MT][NB];
    each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { sum[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
    auto take = [&](const uint4 (&xs)[MT], const uint4 (&as)[NB]) __attribute__((always_inline)) {
      each<0, MT>([&](auto mc) __attribute__((always_inline)) {
        each<0, NB>([&](auto ic) __attribute__((always_inline)) { sum[mc.value][ic.value] = mfma16<BF16>(xs[mc.value], as[ic.value], sum[mc.value][ic.value]); });
      });
    };
    for (int s = begin; s < end; s++) {
      uint4 xs[MT], as[NB];
      each<0, MT>([&](auto mc) __attribute__((always_inline)) { xs[mc.value] = octet(x[mc.value] + 64 * (int64_t)s); });
      each<0, NB>([&](auto ic) __attribute__((always_inline)) { as[ic.value] = octet(a + a_off[ic.value] + 64 * (int64_t)s); });
      take(xs, as);
    }
    if (end_all > whole) {
      const int valid = K - 32 * whole - 8 * g;
      uint4 xs[MT], as[NB];
      each<0, MT>([&](auto mc) __attribute__((always_inline)) { xs[mc.value] = octet_part(x[mc.value] + 64 * (int64_t)whole, valid); });
      each<0, NB>([&](auto ic) __attribute__((always_inline)) { as[ic.value] = octet_part(a + a_off[ic.value] + 64 * (int64_t)whole, valid); });
      take(xs, as);
    }
    each<0, MT * NB * 4>([&](auto ic) __attribute__((always_inline)) {
      constexpr int m = ic.value / (NB * 4), i = ic.value / 4 % NB, r = ic.value % 4;
      acc[m][i][r] = of_sum[m][r] == cur ? sum[m][i][r] : acc[m][i][r];
    });
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

// ---- kernel 2: 16 * MT rows; a wavefront has 64 columns of its own.  The adapter goes in as the first operand: its row m (= lane % 16 of
// the load) of block i is column 16 (m / 4) + 4 i + m % 4, so that a lane's results are 16 neighbouring columns of row lane % 16.
// The rows' v comes through LDS, 128 of the rank at a time: slices added, scaled, in two parts.
template <bool BF16, int MT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p, Shape sh, const float *v) {
  constexpr int CHUNK = 128, PITCH = CHUNK + 8;
  __shared__ __align__(16) uint16_t parts[2][16 * MT][PITCH];
  __shared__ float row_back[16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.y * (16 * MT), col0 = (int64_t)blockIdx.x * 256 + 64 * wave;
  int mine;
  const int n = adapters_of(lane < 16 * MT ? row_id(p, row0 + lane) : -1, mine);
  int id[MT];
  each<0, MT>([&](auto mc) __attribute__((always_inline)) { id[mc.value] = row_id(p, row0 + 16 * mc.value + c); });
  f32x4 acc[MT][4];
  each<0, MT * 4>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / 4][ic.value % 4] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
  int64_t b_off[4];
  each<0, 4>([&](auto ic) __attribute__((always_inline)) {
    const int64_t col = col0 + 16 * (c >> 2) + 4 * ic.value + (c & 3);
    b_off[ic.value] = 2 * ((col < p.outputs ? col : p.outputs - 1) * p.b_col + 8 * g);
  });
  for (int k0 = 0; n && k0 < p.rank; k0 += CHUNK) {
    // sixteen threads per row, eight values each
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = 16 * mc.value + (tid >> 4), k = k0 + 8 * (tid & 15);
      const int of = row_id(p, row0 + r);
      float f[8] = {};
      if (of >= 0 && k < p.rank) {
        const float *at = v + (row0 + r) * sh.pitch_v + k;
        for (int q = 0; q < sh.slices; q++) {
          const float4 a = *(const float4 *)at, b = *(const float4 *)(at + 4);
          f[0] += a.x, f[1] += a.y, f[2] += a.z, f[3] += a.w, f[4] += b.x, f[5] += b.y, f[6] += b.z, f[7] += b.w;
          at += p.tokens * sh.pitch_v;
        }
        const float factor = p.scales ? p.scales[of] : 1.f;
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
    const int steps = (min(CHUNK, p.rank - k0) + 31) / 32;
    if (col0 < p.outputs)
      for (int d = 0; d < n; d++) {
        const int cur = __builtin_amdgcn_readlane(mine, d);
        const char *b = (const char *)p.b + 2 * ((int64_t)cur * p.b_adapter + k0);
        f32x4 sum[MT][4];
        each<0, MT * 4>([&](auto ic) __attribute__((always_inline)) { sum[ic.value / 4][ic.value % 4] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
        for (int s = 0; s < steps; s++) {
          uint4 cols[4];
          each<0, 4>([&](auto ic) __attribute__((always_inline)) { cols[ic.value] = octet_part(b + b_off[ic.value] + 64 * s, p.rank - k0 - 32 * s - 8 * g); });
          each<0, MT>([&](auto mc) __attribute__((always_inline)) {
            constexpr int m = decltype(mc)::value;
            const uint4 hi = *(const uint4 *)&parts[0][16 * m + c][32 * s + 8 * g], lo = *(const uint4 *)&parts[1][16 * m + c][32 * s + 8 * g];
            each<0, 4>([&](auto ic) __attribute__((always_inline)) {
              sum[m][ic.value] = mfma16<BF16>(cols[ic.value], hi, sum[m][ic.value]);
              sum[m][ic.value] = mfma16<BF16>(cols[ic.value], lo, sum[m][ic.value]);
            });
          });
        }
        each<0, MT>([&](auto mc) __attribute__((always_inline)) {
          constexpr int m = decltype(mc)::value;
          const float back = BF16 ? 1.f : row_back[16 * m + c];
          each<0, 4>([&](auto ic) __attribute__((always_inline)) {
            if (id[m] == cur) acc[m][ic.value] += sum[m][ic.value] * back;
          });
        });
      }
    __syncthreads();
  }
  each<0, MT>([&](auto mc) __attribute__((always_inline)) {
    constexpr int m = decltype(mc)::value;
    const int64_t row = row0 + 16 * m + c, col = col0 + 16 * g;
    if (row >= p.tokens || col >= p.outputs) return;
    const uint16_t *base = (const uint16_t *)p.base + row * p.ld_base + col;
    uint16_t *out = (uint16_t *)p.out + row * p.ld_out + col;
    const int have = (int)min((int64_t)16, p.outputs - col);
    uint16_t e[16];
    if (have == 16) __builtin_memcpy(e, base, 32);
    else each<0, 16>([&](auto ic) __attribute__((always_inline)) { e[ic.value] = ic.value < have ? base[ic.value] : 0; });
    if (id[m] >= 0)  // (a row without an adapter is copied as it is)
      each<0, 16>([&](auto ic) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const float was = BF16 ? __uint_as_float((u32)e[i] << 16) : (float)__builtin_bit_cast(_Float16, e[i]);
        const float now = was + acc[m][i / 4][i % 4];
        e[i] = BF16 ? tts_gemm_device::f32_to_bf16(now) : tts_gemm_device::f32_to_f16(now);
      });
    if (have == 16) __builtin_memcpy(out, e, 32);
    else each<0, 16>([&](auto ic) __attribute__((always_inline)) { if (ic.value < have) out[ic.value] = e[ic.value]; });
  });
}

constexpr int CUS = 256;

int row_tile(const LoraParams &p) { return p.tokens <= 1024 ? 16 : 64; }

Shape shape_of(const LoraParams &p) {
  Shape sh;
  const int tile = row_tile(p);
  sh.row_tiles = (int)std::max<int64_t>(1, (p.tokens + tile - 1) / tile);
  // slices of the inputs until there are two workgroups per CU, of at least two steps per wavefront
  const int steps = (int)((p.inputs + 31) / 32);
  sh.slices = std::max(1, std::min({MAX_SLICES, 2 * CUS / sh.row_tiles, steps / 8}));
  sh.pitch_v = (p.rank + 7) & ~7;
  sh.bytes = (size_t)sh.slices * p.tokens * sh.pitch_v * 4;
  return sh;
}

template <bool BF16, int MT>
hipError_t launch_rows(const LoraParams &p, const Shape &sh, hipStream_t s) {
  float *v = (float *)p.workspace;
  const int blocks = (p.rank + 15) / 16;
  auto shrink = [&](auto kernel, int nb) { kernel<<<dim3(sh.row_tiles, sh.slices, (blocks + nb - 1) / nb), 256, 0, s>>>(p, sh, v); };
  if (blocks <= 1) shrink(lora_shrink_kernel<BF16, MT, 1>, 1);
  else if (blocks <= 2) shrink(lora_shrink_kernel<BF16, MT, 2>, 2);
  else shrink(lora_shrink_kernel<BF16, MT, 4>, 4);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  lora_expand_kernel<BF16, MT><<<dim3((unsigned)((p.outputs + 255) / 256), sh.row_tiles), 256, 0, s>>>(p, sh, v);
  return hipGetLastError();
}

}  // namespace

size_t lora_workspace_bytes(const LoraParams &p) { return shape_of(p).bytes; }

hipError_t launch_lora(const LoraParams &p, hipStream_t s) {
  const Shape sh = shape_of(p);
  if (row_tile(p) == 16) return p.bf16 ? launch_rows<true, 1>(p, sh, s) : launch_rows<false, 1>(p, sh, s);
  return p.bf16 ? launch_rows<true, 4>(p, sh, s) : launch_rows<false, 4>(p, sh, s);
}

}  // namespace tts
