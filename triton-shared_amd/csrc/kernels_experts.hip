// The experts of a mixture-of-experts layer for a few tokens: with e = ids[t, j] and f the activation,
//   h[t, j] = f(x[t] Wg[e]) * (x[t] Wu[e])   (or f(x[t] W[e]) without a gate),     y[t] = sum_j weights[t, j] * (h[t, j] Wd[e]).
// At these sizes a picked expert's weights are read for a handful of rows, so their way from memory is all the time there is:
// they are read once, in 16-byte loads, straight into the registers of the matrix instruction; LDS only adds the wavefronts' sums.
//
// Kernel 1, a workgroup per (expert, columns of h): finds the expert's slots (t, j) among the ids, and computes h for them.
// Kernel 2, a workgroup per (expert, columns of y): the slots' share of y, weighted.  Kernel 3 adds a token's slots.
// Both products: 4 wavefronts share k; a step is 32 (or 64) of k against 16 * NB columns.  v_mfma_f32_16x16x32 takes the rows in its
// first operand (lane % 16 the row, lane / 16 the octet of k) and the columns in its second (lane % 16 the column).
//   k contiguous: a lane's octet of a column is one load.
//   columns contiguous: a lane loads NB neighbouring columns of its eight rows of k and puts each column's eight together with
//     v_perm, so that column 8 (lane % 16) + i is lane % 16's of instruction i.
// h stays in 32 bits.  It enters the second product as the sum of two 16-bit values (of bf16: its high half, and the rest
// rounded; of fp16: after scaling its row to below 2^14 by a power of two, since a product of two fp16 sums need not fit fp16), so what is
// rounded is 2^-16 of it: the matrix units wait for memory anyway, and one 16-bit rounding would show as much as the output's own.
#include <cmath>

#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

using namespace row_ops;

// The weights of one step of a wavefront: 16 * NB columns.
//   K1ST: k is contiguous.  OCT octets of k per lane: lane group g = lane / 16 has k STEP s + 8 OCT g ...
template <bool BF16, bool I8, bool K1ST, int NB>
struct Weights {
  static constexpr int ES = I8 ? 1 : 2;
  static constexpr int OCT = K1ST && I8 ? 2 : 1, STEP = 32 * OCT;
  static constexpr int LOADS = K1ST ? NB : 8, DW = K1ST ? 4 : NB * ES / 4;
  Dwords<DW> raw[LOADS];

  // `w`: the step's first k (the same in all lanes); off: the lane's byte offsets (K1ST: of each column's octets; else of its columns
  // in row 8 g); row: the bytes between rows of k; left: how many of k there are from the step's first on
  template <bool TAIL>
  __device__ __forceinline__ void load(const char *w, const u32 *off, int64_t row, int left, int g) {
    each<0, LOADS>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      if constexpr (K1ST) {
        if constexpr (TAIL) raw[i] = load_part<DW, ES>(w + off[i], (left - 8 * OCT * g) * ES);
        else raw[i] = load_dwords<DW>(w + off[i]);
      } else {
        if (!TAIL || 8 * g + i < left) raw[i] = load_dwords<DW>(w + i * row + off[0]);
        else raw[i] = Dwords<DW>{};
      }
    });
  }
  // column block i, octet o: the instruction's operand
  template <int I, int O>
  __device__ __forceinline__ uint4 operand() const {
    u32 v[4];
    each<0, 4>([&](auto pc) __attribute__((always_inline)) {
      constexpr int p = decltype(pc)::value;
      if constexpr (K1ST && !I8) v[p] = raw[I].d[p];
      else if constexpr (K1ST) v[p] = widen_pair<BF16>(__builtin_amdgcn_perm(0, raw[I].d[2 * O + p / 2], p % 2 ? 0x0c030c02 : 0x0c010c00));
      else if constexpr (!I8) v[p] = __builtin_amdgcn_perm(raw[2 * p + 1].d[I / 2], raw[2 * p].d[I / 2], I % 2 ? 0x07060302 : 0x05040100);
      else v[p] = widen_pair<BF16>(__builtin_amdgcn_perm(raw[2 * p + 1].d[I / 4], raw[2 * p].d[I / 4], 0x0c040c00 + (I % 4) * 0x00010001));
    });
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
};

// The rows' side of a step, in 16-bit elements: one operand per octet
template <int OCT>
struct Rows16 {
  static constexpr int PARTS = 1;
  uint4 v[OCT];
  template <bool TAIL>
  __device__ __forceinline__ void load(const char *row, int k, int left, int g) {  // k: the lane's first
    each<0, OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      Dwords<4> d;
      if constexpr (TAIL) d = load_part<4, 2>(row + 2 * (int64_t)(k + 8 * o), 2 * (left - 8 * OCT * g - 8 * o));
      else d = load_dwords<4>(row + 2 * (int64_t)(k + 8 * o));
      v[o] = make_uint4(d.d[0], d.d[1], d.d[2], d.d[3]);
    });
  }
  template <int O, int PART>
  __device__ __forceinline__ uint4 operand(float) const { return v[O]; }
};

// ... in 32 bits, 16-byte aligned, padded with anything up to a multiple of 8; two operands per octet, the high part and the rest
template <bool BF16, int OCT>
struct Rows32 {
  static constexpr int PARTS = 2;
  float v[OCT][8];
  template <bool TAIL>
  __device__ __forceinline__ void load(const char *row, int k, int left, int g) {
    each<0, OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      const int have = left - 8 * OCT * g - 8 * o;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (!TAIL || have > 0) {
        const float4 *q = (const float4 *)(row + 4 * (int64_t)(k + 8 * o));
        a = q[0], b = q[1];
      }
      const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      each<0, 8>([&](auto ic) __attribute__((always_inline)) { v[o][ic.value] = TAIL && ic.value >= have ? 0.f : f[ic.value]; });
    });
  }
  template <int O, int PART>
  __device__ __forceinline__ uint4 operand(float scale) const {
    return split_part<BF16, PART>(v[O], scale);
  }
};

// acc[m][i] += rows 16 m ... times column block i, over this wavefront's share of k's steps.
//   w: the expert's matrix (all lanes the same), off and row as in Weights; rows[m]: the lane's row
template <bool BF16, int MT, int NB, class W, class R>
__device__ __forceinline__ void product(f32x4 (&acc)[MT][NB], const char *w, const u32 *off, int64_t w_k, const char *const (&rows)[MT], const float (&scale)[MT], int64_t K,
                                        int wave, int g) {
  constexpr int U = W::DW * W::LOADS > 16 ? 2 : 4;  // steps in flight
  const int steps = (int)((K + W::STEP - 1) / W::STEP), whole = (int)(K / W::STEP);
  const int begin = (int)((int64_t)wave * steps / 4), end_all = (int)((int64_t)(wave + 1) * steps / 4), end = end_all < whole ? end_all : whole;
  const int64_t step_bytes = w_k * W::STEP;
  W ring[U];
  R rring[U][MT];
  auto take = [&](W &wt, R (&rt)[MT]) __attribute__((always_inline)) {
    each<0, W::OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      uint4 a[MT][R::PARTS];
      each<0, MT>([&](auto mc) __attribute__((always_inline)) {
        each<0, R::PARTS>([&](auto pc) __attribute__((always_inline)) { a[mc.value][pc.value] = rt[mc.value].template operand<o, decltype(pc)::value>(scale[mc.value]); });
      });
      each<0, NB>([&](auto ic) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const uint4 b = wt.template operand<i, o>();
        each<0, MT>([&](auto mc) __attribute__((always_inline)) {
          each<0, R::PARTS>([&](auto pc) __attribute__((always_inline)) { acc[mc.value][i] = mfma16<BF16>(a[mc.value][pc.value], b, acc[mc.value][i]); });
        });
      });
    });
  };
  if (begin < end) {
    auto fetch = [&](int s, W &wt, R (&rt)[MT]) __attribute__((always_inline)) {
      const int at = s < end ? s : end - 1;  // (loads past the last step fetch it again, and nobody takes them)
      wt.template load<false>(w + at * step_bytes, off, w_k, 0, g);
      each<0, MT>([&](auto mc) __attribute__((always_inline)) { rt[mc.value].template load<false>(rows[mc.value], at * W::STEP + 8 * W::OCT * g, 0, g); });
    };
    each<0, U>([&](auto uc) __attribute__((always_inline)) { fetch(begin + uc.value, ring[uc.value], rring[uc.value]); });
    int s = begin;
    for (; s + U <= end; s += U)
      each<0, U>([&](auto uc) __attribute__((always_inline)) {
        take(ring[uc.value], rring[uc.value]);
        fetch(s + U + uc.value, ring[uc.value], rring[uc.value]);
      });
    each<0, U>([&](auto uc) __attribute__((always_inline)) {
      if (s + uc.value < end) take(ring[uc.value], rring[uc.value]);
    });
  }
  if (end_all > whole) {  // the part step
    const int left = (int)(K - (int64_t)whole * W::STEP);
    ring[0].template load<true>(w + whole * step_bytes, off, w_k, left, g);
    each<0, MT>([&](auto mc) __attribute__((always_inline)) { rring[0][mc.value].template load<true>(rows[mc.value], whole * W::STEP + 8 * W::OCT * g, left, g); });
    take(ring[0], rring[0]);
  }
}

// The expert of this workgroup and its slots among ids[0 .. slots): in ascending order in `list`; returns their number.  With as
// many groups of workgroups as experts, group y has expert y; with fewer, it has that of slot y, if no slot before has it.
__device__ __forceinline__ int slots_of_expert(const ExpertsParams &p, int y, bool by_slot, uint16_t *list, int *counts, int &expert) {
  const int slots = (int)p.tokens * p.top;
  auto id_of = [&](int slot) __attribute__((always_inline)) {
    const u32 t = (u32)slot / (u32)p.top;
    return p.ids[(int64_t)t * p.ld_ids + (slot - (int)t * p.top)];
  };
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  expert = by_slot ? __builtin_amdgcn_readfirstlane(id_of(y)) : y;
  if ((u32)expert >= (u32)p.experts) return 0;
  // wavefront w has the w'th quarter of the slots (in whole 64s)
  constexpr int MOST = EXPERTS_MAX_SLOTS / 256;
  const int per = (slots + 255) / 256;
  uint64_t match[MOST];
  int mine = 0, before = 0;
  for (int i = 0; i < MOST; i++) {
    match[i] = 0;
    if (i < per) {
      const int slot = (wave * per + i) * 64 + lane;
      match[i] = __ballot(slot < slots && id_of(slot < slots ? slot : 0) == expert);
      mine += __popcll(match[i]);
      const int bound = y - (wave * per + i) * 64;  // slots before y
      if (by_slot && bound > 0) before |= (match[i] & (bound >= 64 ? ~0ull : (1ull << bound) - 1)) != 0;
    }
  }
  if (lane == 0) counts[wave] = mine | before << 16;
  __syncthreads();
  int at = 0, all = 0, seen = 0;
  for (int w = 0; w < 4; w++) {
    const int c = counts[w];
    if (w < wave) at += c & 0xffff;
    all += c & 0xffff;
    seen |= c >> 16;
  }
  if (seen) return 0;
  for (int i = 0; i < MOST; i++)
    if (i < per) {
      const int lower = __popcll(match[i] & ((1ull << lane) - 1));
      if (match[i] >> lane & 1) list[at + lower] = (uint16_t)((wave * per + i) * 64 + lane);
      at += __popcll(match[i]);
    }
  __syncthreads();
  return all;
}

// The wavefronts' sums of rows 16 m ..: to LDS, in the order of columns; a row's 16 * NB columns are PITCH floats apart
template <bool K1ST, int NB, int PITCH>
__device__ __forceinline__ void put_sums(float *red, const f32x4 (&acc)[NB], int wave, int lane) {
  const int c = lane & 15, g = lane >> 4;
  each<0, NB>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    const int col = K1ST ? 16 * i + c : NB * c + i;
    each<0, 4>([&](auto rc) __attribute__((always_inline)) { red[(wave * 16 + 4 * g + rc.value) * PITCH + col] = acc[i][rc.value]; });
  });
}

__device__ __forceinline__ float activate(int kind, float v) {
  if (kind == ACT_SILU) return v / (1.f + expf(-v));
  if (kind == ACT_RELU) return v < 0.f ? 0.f : v;
  // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u))
  const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
  return v / (1.f + expf(-2.f * u));
}

struct Layout {  // of the workspace
  int64_t pitch_h;     // floats between slots' rows of h
  int slabs;           // of columns of h
  float *h, *row_max, *partial;
  size_t bytes;
};

template <int NB>
constexpr int COLS = 16 * NB;

Layout layout_of(const ExpertsParams &p, int h_cols) {
  Layout l;
  const int64_t slots = p.tokens * p.top;
  l.pitch_h = (p.inner + 7) & ~(int64_t)7;
  l.slabs = (int)((p.inner + h_cols - 1) / h_cols);
  const size_t h = (size_t)slots * l.pitch_h * 4, most = ((size_t)slots * l.slabs * 4 + 255) & ~(size_t)255, part = (size_t)slots * p.outputs * 4;
  char *base = (char *)p.workspace;
  l.h = (float *)base;
  l.row_max = (float *)(base + ((h + 255) & ~(size_t)255));
  l.partial = (float *)((char *)l.row_max + most);
  l.bytes = ((h + 255) & ~(size_t)255) + most + part;
  return l;
}

// ---- kernel 1
template <bool BF16, bool I8, bool K1ST, bool GATED, int MT, int NB>
__global__ __launch_bounds__(256) void experts_up_kernel(ExpertsParams p, Layout l, int by_slot) {
  using W = Weights<BF16, I8, K1ST, NB>;
  using R = Rows16<W::OCT>;
  constexpr int HC = GATED ? COLS<NB> / 2 : COLS<NB>, PITCH = COLS<NB> + 4;  // columns of h
  __shared__ uint16_t list[EXPERTS_MAX_SLOTS];
  __shared__ int counts[4];
  __shared__ float red[4 * 16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  int expert;
  const int n = slots_of_expert(p, blockIdx.y, by_slot, list, counts, expert);
  if (n == 0) return;
  const int inner = (int)p.inner, c0 = blockIdx.x * HC;
  // Columns past the last are other columns' again: whoever computes one twice gets the same.
  u32 off[K1ST ? NB : 1];
  if constexpr (K1ST)
    each<0, NB>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, in_half = GATED ? i % (NB / 2) : i;
      const int col = min(c0 + 16 * in_half + c, inner - 1) + (GATED && i >= NB / 2 ? inner : 0);
      off[i] = (u32)((col * p.up.w_n + 8 * W::OCT * g) * W::ES);
    });
  else {
    const int col = min(c0 + NB * (GATED ? c % 8 : c), inner - NB) + (GATED && c >= 8 ? inner : 0);
    off[0] = (u32)((8 * g * p.up.w_k + col) * W::ES);
  }
  const char *w = (const char *)p.up.w + (int64_t)expert * p.up.w_expert * W::ES;
  const float *scales = I8 ? p.up.scale + (int64_t)expert * p.up.scale_expert : nullptr;
  const float one[MT] = {};
  for (int r0 = 0; r0 < n; r0 += 16 * MT) {
    const char *rows[MT];
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = min(r0 + 16 * mc.value + c, n - 1);
      rows[mc.value] = (const char *)p.x + (int64_t)((u32)list[r] / (u32)p.top) * p.ld_x * 2;
    });
    f32x4 acc[MT][NB];
    each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
    product<BF16, MT, NB, W, R>(acc, w, off, p.up.w_k * W::ES, rows, one, p.hidden, wave, g);
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      if (r0 + 16 * m >= n) return;
      put_sums<K1ST, NB, PITCH>(red, acc[m], wave, lane);
      __syncthreads();
      // 16 threads per row
      const int r = tid >> 4, part = tid & 15;
      const int slot = r0 + 16 * m + r < n ? list[r0 + 16 * m + r] : -1;
      float most = 0.f;
      for (int j = part; j < HC; j += 16) {
        // the column that place j holds
        const int col = K1ST ? min(c0 + j, inner - 1) : min(c0 + j / NB * NB, inner - NB) + j % NB;
        float gate = 0.f, up = 0.f;
        for (int q = 0; q < 4; q++) {
          gate += red[(q * 16 + r) * PITCH + j];
          if (GATED) up += red[(q * 16 + r) * PITCH + HC + j];
        }
        if (I8) {
          gate *= scales[col];
          if (GATED) up *= scales[inner + col];
        }
        const float h = GATED ? activate(p.activation, gate) * up : activate(p.activation, gate);
        most = fmaxf(most, fabsf(h));
        if (slot >= 0) l.h[slot * l.pitch_h + col] = h;
      }
      if (!BF16) {
        for (int d = 1; d < 16; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        if (slot >= 0 && part == 0) l.row_max[(int64_t)slot * l.slabs + blockIdx.x] = most;
      }
      __syncthreads();
    });
  }
}

// ---- kernel 2
template <bool BF16, bool I8, bool K1ST, int MT, int NB>
__global__ __launch_bounds__(256) void experts_down_kernel(ExpertsParams p, Layout l, int by_slot) {
  using W = Weights<BF16, I8, K1ST, NB>;
  using R = Rows32<BF16, W::OCT>;
  constexpr int PITCH = COLS<NB> + 4;
  __shared__ uint16_t list[EXPERTS_MAX_SLOTS];
  __shared__ int counts[4];
  __shared__ float red[4 * 16 * PITCH];
  __shared__ float row_scale[16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  int expert;
  const int n = slots_of_expert(p, blockIdx.y, by_slot, list, counts, expert);
  if (n == 0) return;
  const int outputs = (int)p.outputs, c0 = blockIdx.x * COLS<NB>;
  u32 off[K1ST ? NB : 1];
  if constexpr (K1ST)
    each<0, NB>([&](auto ic) __attribute__((always_inline)) { off[ic.value] = (u32)((min(c0 + 16 * ic.value + c, outputs - 1) * p.down.w_n + 8 * W::OCT * g) * W::ES); });
  else
    off[0] = (u32)((8 * g * p.down.w_k + min(c0 + NB * c, outputs - NB)) * W::ES);
  const char *w = (const char *)p.down.w + (int64_t)expert * p.down.w_expert * W::ES;
  const float *scales = I8 ? p.down.scale + (int64_t)expert * p.down.scale_expert : nullptr;
  for (int r0 = 0; r0 < n; r0 += 16 * MT) {
    const char *rows[MT];
    float scale[MT];
    if (!BF16) {  // 2^-e with the row's largest |h| 2^-e in [2^13, 2^14)
      for (int r = tid >> 4; r < 16 * MT; r += 16) {
        float most = 0.f;
        if (r0 + r < n)
          for (int j = tid & 15; j < l.slabs; j += 16) most = fmaxf(most, l.row_max[(int64_t)list[r0 + r] * l.slabs + j]);
        for (int d = 1; d < 16; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        if ((tid & 15) == 0) row_scale[r] = fp16_scale(most);
      }
      __syncthreads();
    }
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = min(r0 + 16 * mc.value + c, n - 1);
      rows[mc.value] = (const char *)(l.h + list[r] * l.pitch_h);
      scale[mc.value] = BF16 ? 1.f : row_scale[r - r0];
    });
    f32x4 acc[MT][NB];
    each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
    product<BF16, MT, NB, W, R>(acc, w, off, p.down.w_k * W::ES, rows, scale, p.inner, wave, g);
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      if (r0 + 16 * m >= n) return;
      put_sums<K1ST, NB, PITCH>(red, acc[m], wave, lane);
      __syncthreads();
      const int r = tid >> 4;
      if (r0 + 16 * m + r < n) {
        const int slot = list[r0 + 16 * m + r];
        const u32 t = (u32)slot / (u32)p.top;
        const float weight = p.weights[(int64_t)t * p.ld_weights + (slot - (int)t * p.top)];
        const float back = BF16 ? 1.f : 1.f / row_scale[16 * m + r];  // (a power of two)
        for (int j = tid & 15; j < COLS<NB>; j += 16) {
          const int col = K1ST ? min(c0 + j, outputs - 1) : min(c0 + j / NB * NB, outputs - NB) + j % NB;
          float v = 0.f;
          for (int q = 0; q < 4; q++) v += red[(q * 16 + r) * PITCH + j];
          if (!BF16) v *= back;
          if (I8) v *= scales[col];
          l.partial[(int64_t)slot * outputs + col] = v * weight;
        }
      }
      __syncthreads();
    });
  }
}

// ---- kernel 3: y[t] = the sum of its slots
template <bool BF16>
__global__ __launch_bounds__(256) void experts_sum_kernel(ExpertsParams p, const float *partial) {
  const int64_t t = blockIdx.y, col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.outputs) return;
  float v = 0.f;
  for (int j = 0; j < p.top; j++)
    if ((u32)p.ids[t * p.ld_ids + j] < (u32)p.experts) v += partial[(t * p.top + j) * p.outputs + col];
  ((uint16_t *)p.out)[t * p.ld_out + col] = BF16 ? tts_gemm_device::f32_to_bf16(v) : tts_gemm_device::f32_to_f16(v);
}

constexpr int NB_UP = 8, NB_DOWN = 8;

int h_cols(const ExpertsParams &p) { return p.gated ? 8 * NB_UP : 16 * NB_UP; }

template <bool BF16, bool I8>
hipError_t launch_typed(const ExpertsParams &p, hipStream_t s) {
  const Layout l = layout_of(p, h_cols(p));
  const int64_t slots = p.tokens * p.top;
  const int by_slot = slots < p.experts, groups = by_slot ? (int)slots : p.experts;
  const bool wide = p.tokens > 16;
  auto up = [&](auto k1st, auto gated, auto mt) {
    experts_up_kernel<BF16, I8, decltype(k1st)::value != 0, decltype(gated)::value != 0, decltype(mt)::value, NB_UP><<<dim3(l.slabs, groups), 256, 0, s>>>(p, l, by_slot);
    return hipGetLastError();
  };
  auto down = [&](auto k1st, auto mt) {
    experts_down_kernel<BF16, I8, decltype(k1st)::value != 0, decltype(mt)::value, NB_DOWN>
        <<<dim3((unsigned)((p.outputs + 16 * NB_DOWN - 1) / (16 * NB_DOWN)), groups), 256, 0, s>>>(p, l, by_slot);
    return hipGetLastError();
  };
  auto with_rows = [&](auto mt) {
    const hipError_t e = p.up.w_k == 1 ? (p.gated ? up(Int<1>{}, Int<1>{}, mt) : up(Int<1>{}, Int<0>{}, mt)) : (p.gated ? up(Int<0>{}, Int<1>{}, mt) : up(Int<0>{}, Int<0>{}, mt));
    if (e != hipSuccess) return e;
    return p.down.w_k == 1 ? down(Int<1>{}, mt) : down(Int<0>{}, mt);
  };
  const hipError_t e = wide ? with_rows(Int<2>{}) : with_rows(Int<1>{});
  if (e != hipSuccess) return e;
  experts_sum_kernel<BF16><<<dim3((unsigned)((p.outputs + 255) / 256), (unsigned)p.tokens), 256, 0, s>>>(p, l.partial);
  return hipGetLastError();
}

}  // namespace

size_t experts_workspace_bytes(const ExpertsParams &p) { return layout_of(p, h_cols(p)).bytes; }

hipError_t launch_experts(const ExpertsParams &p, hipStream_t s) {
  if (p.bf16) return p.int8 ? launch_typed<true, true>(p, s) : launch_typed<true, false>(p, s);
  return p.int8 ? launch_typed<false, true>(p, s) : launch_typed<false, false>(p, s);
}

}  // namespace tts
