// The experts of a mixture-of-experts layer for a few tokens: with e = ids[t, j] and f the activation,
//   h[t, j] = f(x[t] Wg[e]) * (x[t] Wu[e])   (or f(x[t] W[e]) without a gate),     y[t] = sum_j weights[t, j] * (h[t, j] Wd[e]).
// At these sizes a picked expert's weights are read for a handful of rows, so their way from memory is what there is to spend:
// they are read once, in 16-byte loads, straight into the registers of the matrix instruction; LDS only adds the wavefronts' sums.
//
// Kernel 1, a workgroup per (expert, columns of h): finds the expert's slots (t, j) among the ids, and computes h for them.
// Kernel 2, a workgroup per (expert, columns of y): the slots' share of y, weighted, in 32 bits.  Kernel 3 adds a token's slots, in their order.
// Both products: 4 wavefronts share k.  v_mfma_f32_16x16x32 takes 16 rows in its first operand (lane % 16 the row, lane / 16 the octet
// of k) and 16 columns in its second; how the weights get there is told at `Weights`.  Rows (of x, of h) come straight from the caches into
// the first operand, asked for two steps ahead of the weights' one.
// h enters the second product as the sum of two 16-bit values (bf16: its high half, and the rest rounded, by kernel 1;
// fp16: by kernel 2, after scaling its row to below 2^14 by a power of two, since a product of two fp16 sums need not fit fp16), so what is
// rounded is 2^-16 of it: one 16-bit rounding would show as much as the output's own.
//
// What bounds it: large weights, the way from memory (4 tokens, 6 of 8 experts of 4096 x 8192, fp16: kernel 1 reads 805 MB in 155 us, 5.2 TB/s); with
// many rows per expert also the rows' way from L2, which shares the path to the CU with the weights (a probe that reads weights in this
// pattern reaches 6.3 TB/s, with half as many row loads beside them 5.4, with as many 4.1): 256 tokens, 64 experts of 4096 x 1536, kernel 1
// 5.2 TB/s, kernel 2, whose rows are two parts, 3.6.  One token: three launches and the chain id - rows - weights - sums in each, 15 + 9.5 + 4 us.
#include <algorithm>
#include <cmath>

#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

using namespace row_ops;

// The weights of one step of a wavefront: 16 * NB columns, in groups of GROUP neighbours.  A step is 32 * OCT of k, of which lane group g = lane / 16
// multiplies 8 * OCT g ..: operand o of a column block has octet OCT g + o in that group.
//   k contiguous: a load takes the 128 bytes of k that a step is from 8 columns, lane % 8 the column, lane / 8 the sixteenth byte: whole
//     cache lines, since what a load leaves of a line may be gone before the next load asks for it.  Of two
//     loads X and Y, columns 0-7 and 8-15 of a block, lanes c < 8 of X hold chunk 2 g of column c and lanes c >= 8 chunk 2 g + 1 of
//     column c - 8, and Y likewise: exchanging halves of 16 lanes (one DPP move per dword) gives all columns chunk 2 g, or 2 g + 1.
//   columns contiguous: a lane loads NB neighbouring columns of its eight rows of k, and puts each column's eight together with v_perm.
template <bool BF16, bool I8, bool K1ST, int NB>
struct Weights {
  static constexpr int ES = I8 ? 1 : 2;
  static constexpr int OCT = !K1ST ? 1 : I8 ? 4 : 2, STEP = 32 * OCT, LANE = 8 * OCT, GROUP = K1ST ? 8 : NB;
  static constexpr int LOADS = K1ST ? 2 * NB : 8, DW = K1ST ? 4 : NB * ES / 4;
  Dwords<DW> raw[LOADS];

  // where a group's columns begin in its half of the tile (GATED: the first half of the groups is the gate's); groups past the last column
  // are the last GROUP columns again: whoever computes one twice gets the same
  static __device__ __forceinline__ int column(int c0, int group, int columns) { return min(c0 + group * GROUP, columns - GROUP); }
  // a lane's bytes from the first of its group's columns (k contiguous), or from the matrix's first
  static __device__ __forceinline__ u32 lane_offset(int lane, int64_t w_k, int64_t w_n, int column) {
    return K1ST ? (u32)((lane & 7) * w_n * ES + 16 * (lane >> 3)) : (u32)((8 * (lane >> 4) * w_k + column) * ES);
  }
  // load I of a step.  `w`: the step's first k; at(j): the first of group j's columns (k contiguous)
  template <int I, class F>
  __device__ __forceinline__ void load(const char *w, u32 off, int64_t w_k, int64_t w_n, F &&at) {
    asm("" : "+v"(off));  // (seen as a 32-bit value here, it goes into the load: scalar base, vector offset)
    if constexpr (K1ST) raw[I] = stream_dwords<DW>(w + at(I) * (w_n * ES) + off);
    else raw[I] = stream_dwords<DW>(w + I * (w_k * ES) + off);
  }
  // what block I needs of a part step of which `left` of k are there
  template <int I, class F>
  __device__ __forceinline__ void load_part_of(const char *w, u32 off, int64_t w_k, int64_t w_n, F &&at, int left, int lane) {
    if constexpr (K1ST)
      each<2 * I, 2 * I + 2>([&](auto jc) __attribute__((always_inline)) { raw[jc.value] = load_part(w + at(jc.value) * (w_n * ES) + off, left * ES - 16 * (lane >> 3)); });
    else if constexpr (I == 0)
      each<0, 8>([&](auto jc) __attribute__((always_inline)) {
        if (8 * (lane >> 4) + jc.value < left) raw[jc.value] = load_dwords<DW>(w + jc.value * (w_k * ES) + off);
        else raw[jc.value] = Dwords<DW>{};
      });
  }
  // dword d of chunk 2 g + HALF of the columns of block I
  template <int I, int HALF, int D>
  __device__ __forceinline__ u32 chunk() const {
    const int x = raw[2 * I].d[D], y = raw[2 * I + 1].d[D];
    return HALF == 0 ? __builtin_amdgcn_update_dpp(x, y, 0x128, 0xf, 0xc, false) : __builtin_amdgcn_update_dpp(y, x, 0x128, 0xf, 0x3, false);  // row_ror:8 into lanes 8-15, or 0-7
  }
  // column block I, octet O: the instruction's operand
  template <int I, int O>
  __device__ __forceinline__ uint4 operand() const {
    u32 v[4];
    each<0, 4>([&](auto pc) __attribute__((always_inline)) {
      constexpr int p = decltype(pc)::value;
      if constexpr (K1ST && !I8) v[p] = chunk<I, O, p>();
      else if constexpr (K1ST) v[p] = widen_pair<BF16>(__builtin_amdgcn_perm(0, chunk<I, O / 2, 2 * (O % 2) + p / 2>(), p % 2 ? 0x0c030c02 : 0x0c010c00));
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
  __device__ __forceinline__ void load(const char *row, int64_t, int64_t k, int left, int g) {  // k: the lane's first
    each<0, OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      Dwords<4> d;
      if constexpr (TAIL) d = load_part(row + 2 * (int64_t)(k + 8 * o), 2 * (left - 8 * OCT * g - 8 * o));
      else d = load_dwords<4>(row + 2 * (int64_t)(k + 8 * o));
      v[o] = make_uint4(d.d[0], d.d[1], d.d[2], d.d[3]);
    });
  }
  template <int O, int PART>
  __device__ __forceinline__ uint4 operand(float) const { return v[O]; }
};

// ... of h: two operands per octet, the high part and the rest.  Rows are 16-byte aligned and end with zeros up to a multiple of 8.
//   bf16: kernel 1 has left the two parts, `plane` bytes apart;  fp16: the 32 bits, which are split here, after scaling
template <bool BF16, int OCT>
struct RowsOfH {
  static constexpr int PARTS = 2;
  uint4 v[OCT][2];
  template <bool TAIL>
  __device__ __forceinline__ void load(const char *row, int64_t plane, int64_t k, int left, int g) {
    each<0, OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      if (!TAIL || left - 8 * OCT * g - 8 * o > 0) {
        const char *q = row + (BF16 ? 2 : 4) * (int64_t)(k + 8 * o);
        v[o][0] = *(const uint4 *)q;
        v[o][1] = *(const uint4 *)(q + (BF16 ? plane : 16));
      } else
        v[o][0] = v[o][1] = make_uint4(0, 0, 0, 0);
    });
  }
  template <int O, int PART>
  __device__ __forceinline__ uint4 operand(float scale) const {
    if constexpr (BF16) return v[O][PART];
    else {
      const uint4 a = v[O][0], b = v[O][1];
      const float f[8] = {__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w),
                          __uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w)};
      return split_part<false, PART>(f, scale);
    }
  }
};

// This wavefront's share of k's steps: acc[m][i] += rows 16 m ... times column block i.  `begin` sends the first steps' weights on their way, which
// needs the expert alone; `rows` takes the rows when they are known.
template <bool BF16, int NB, int WAVES, class W, class At>
struct Product {
  static constexpr int U = W::DW * W::LOADS > 16 ? 1 : 2;  // steps in flight
  const char *w;       // the expert's matrix (all lanes the same); off, w_k, w_n, at: as in Weights
  const int64_t w_k, w_n, K;
  u32 off;
  At at;
  const int lane, g;
  int first, end, whole, part;
  const char *next;    // the step that is fetched next, and how many there are from it on
  int ahead;
  W ring[U];

  __device__ __forceinline__ Product(const ExpertMatrix &m, int expert, int64_t K_, At at_, int wave, int lane_)
      : w((const char *)m.w + (int64_t)expert * m.w_expert * W::ES), w_k(m.w_k), w_n(m.w_n), K(K_), at(at_), lane(lane_), g(lane_ >> 4) {
    const int steps = (int)((K + W::STEP - 1) / W::STEP);
    whole = (int)(K / W::STEP);
    first = (int)((int64_t)wave * steps / WAVES);
    const int last = (int)((int64_t)(wave + 1) * steps / WAVES);
    end = last < whole ? last : whole;
    part = last > whole;
  }
  __device__ __forceinline__ void fetch(W &wt) {  // (past the last: the last again, and nobody takes it)
    each<0, W::LOADS>([&](auto ic) __attribute__((always_inline)) { wt.template load<ic.value>(next, off, w_k, w_n, at); });
    next += --ahead > 0 ? w_k * (W::STEP * W::ES) : 0;
  }
  __device__ __forceinline__ void begin(int c0) {  // with the columns from c0 on
    at.c0 = c0;
    off = W::lane_offset(lane, w_k, w_n, at(lane & 15));
    next = w + first * (w_k * (W::STEP * W::ES));
    ahead = end - first;
    if (first < end) each<0, U>([&](auto uc) __attribute__((always_inline)) { fetch(ring[uc.value]); });
  }
  // column blocks I and I + 1, whose sums take turns: a matrix instruction waits for the one before that adds to the same
  template <int I, class R, int MT>
  __device__ __forceinline__ void take_blocks(f32x4 (&acc)[MT][NB], const W &wt, const uint4 (&a)[W::OCT][MT][R::PARTS]) {
    each<0, W::OCT>([&](auto oc) __attribute__((always_inline)) {
      constexpr int o = decltype(oc)::value;
      const uint4 b[2] = {wt.template operand<I, o>(), wt.template operand<I + 1, o>()};
      each<0, R::PARTS>([&](auto pc) __attribute__((always_inline)) {
        each<0, 2 * MT>([&](auto nc) __attribute__((always_inline)) {
          constexpr int m = decltype(nc)::value / 2, i = decltype(nc)::value % 2;
          acc[m][I + i] = mfma16<BF16>(a[o][m][pc.value], b[i], acc[m][I + i]);
        });
      });
    });
    __builtin_amdgcn_sched_barrier(0);  // (not more at a time: their operands would take the registers of wavefronts that could run)
  }
  template <class R, int MT>
  __device__ __forceinline__ void operands(uint4 (&a)[W::OCT][MT][R::PARTS], const R (&rt)[MT], const float (&scale)[MT]) {
    each<0, W::OCT * MT * R::PARTS>([&](auto nc) __attribute__((always_inline)) {
      constexpr int n = decltype(nc)::value, o = n / (MT * R::PARTS), m = n / R::PARTS % MT, part = n % R::PARTS;
      a[o][m][part] = rt[m].template operand<o, part>(scale[m]);
    });
  }
  template <class R, int MT>
  __device__ __forceinline__ void take(f32x4 (&acc)[MT][NB], const W &wt, const R (&rt)[MT], const float (&scale)[MT]) {
    uint4 a[W::OCT][MT][R::PARTS];
    operands<R, MT>(a, rt, scale);
    each<0, NB / 2>([&](auto ic) __attribute__((always_inline)) { take_blocks<2 * ic.value, R, MT>(acc, wt, a); });
  }
  template <class R, int MT>
  __device__ __forceinline__ void rows(f32x4 (&acc)[MT][NB], const char *const (&row)[MT], int64_t plane, const float (&scale)[MT]) {
    constexpr int RU = MT > 2 ? 1 : 2, TURN = U > RU ? U : RU;  // rows are asked for two steps ahead, so that nothing waits for them behind the weights
    R rring[RU][MT];
    if (first < end) {
      int64_t k = first * W::STEP + W::LANE * g;  // the lane's first k of the rows' next step
      int rows_ahead = end - first;
      auto fetch_rows = [&](R (&rt)[MT]) __attribute__((always_inline)) {
        each<0, MT>([&](auto mc) __attribute__((always_inline)) { rt[mc.value].template load<false>(row[mc.value], plane, k, 0, g); });
        k += --rows_ahead > 0 ? W::STEP : 0;
      };
      each<0, RU>([&](auto uc) __attribute__((always_inline)) { fetch_rows(rring[uc.value]); });
      int s = first;
      auto turn = [&]() __attribute__((always_inline)) {
        each<0, TURN>([&](auto uc) __attribute__((always_inline)) {
          take<R, MT>(acc, ring[uc.value % U], rring[uc.value % RU], scale);
          __builtin_amdgcn_sched_barrier(0);  // (the next loads go to the registers that are free now, not to others before)
          fetch(ring[uc.value % U]);
          fetch_rows(rring[uc.value % RU]);
          __builtin_amdgcn_sched_barrier(0);
        });
        s += TURN;
      };
      // The first turn's loads were sent in another order, weights before rows.  It has to be outside of the loop: the loop waits for counts
      // of loads in flight, which are those of the order that leaves the fewest.
      if (s + TURN <= end) {
        turn();
        while (s + TURN <= end) turn();
      }
      each<0, TURN>([&](auto uc) __attribute__((always_inline)) {
        if (s + uc.value < end) {
          take<R, MT>(acc, ring[uc.value % U], rring[uc.value % RU], scale);
          if (uc.value + U < TURN) fetch(ring[uc.value % U]);
          if (uc.value + RU < TURN) fetch_rows(rring[uc.value % RU]);
        }
      });
    }
    if (part) {  // the last, part step
      const int left = (int)(K - (int64_t)whole * W::STEP);
      const char *at_w = w + whole * (w_k * (W::STEP * W::ES));
      each<0, MT>([&](auto mc) __attribute__((always_inline)) { rring[0][mc.value].template load<true>(row[mc.value], plane, whole * W::STEP + W::LANE * g, left, g); });
      uint4 a[W::OCT][MT][R::PARTS];
      operands<R, MT>(a, rring[0], scale);
      each<0, NB / 2>([&](auto ic) __attribute__((always_inline)) {
        ring[0].template load_part_of<2 * ic.value>(at_w, off, w_k, w_n, at, left, lane);
        ring[0].template load_part_of<2 * ic.value + 1>(at_w, off, w_k, w_n, at, left, lane);
        take_blocks<2 * ic.value, R, MT>(acc, ring[0], a);
      });
    }
  }
};

// Which expert group y of the workgroups has: with as many groups as experts, the y'th; with fewer, that of slot y (and SlotsOf
// finds out whether a slot before has it).
__device__ __forceinline__ int id_of(const ExpertsParams &p, int slot) {
  if (p.ld_ids == p.top) return p.ids[slot];
  const u32 t = (u32)slot / (u32)p.top;
  return p.ids[(int64_t)t * p.ld_ids + (slot - (int)t * p.top)];
}
__device__ __forceinline__ int expert_of(const ExpertsParams &p, int y, bool by_slot) { return by_slot ? __builtin_amdgcn_readfirstlane(id_of(p, y)) : y; }

// The expert's slots among ids[0 .. slots).  `ask` sends for the ids, before the weights do: loads come back in order.
template <int WAVES>
struct SlotsOf {
  static constexpr int MOST = EXPERTS_MAX_SLOTS / (64 * WAVES);
  int slots, per, id[MOST];
  __device__ __forceinline__ void ask(const ExpertsParams &p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    slots = (int)p.tokens * p.top;
    // wavefront w has the w'th part of the slots (in whole 64s), of 64 slots or fewer each has them all
    per = (slots + 64 * WAVES - 1) / (64 * WAVES);
    each<0, MOST / 4>([&](auto jc) __attribute__((always_inline)) {
      constexpr int j = 4 * decltype(jc)::value;
      if (j < per)
        each<0, 4>([&](auto ic) __attribute__((always_inline)) { id[j + ic.value] = id_of(p, min(((slots <= 64 ? 0 : wave * per) + j + ic.value) * 64 + lane, slots - 1)); });
    });
  }
  // in ascending order in `list`; returns their number, or 0 where another group has the expert (by_slot: a slot before y)
  __device__ __forceinline__ int find(int expert, int y, bool by_slot, uint16_t *list, int *counts) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (slots <= 64) {  // every wavefront finds, and writes, the same
      const uint64_t match = __ballot(lane < slots && id[0] == expert);
      if (by_slot && (match & ((1ull << y) - 1))) return 0;
      if (match >> lane & 1) list[__popcll(match & ((1ull << lane) - 1))] = (uint16_t)lane;
      __builtin_amdgcn_wave_barrier();
      return __popcll(match);
    }
    uint64_t match[MOST];
    int mine = 0, before = 0;
    each<0, MOST>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      match[i] = 0;
      if (i / 4 * 4 < per) {
        const int slot = (wave * per + i) * 64 + lane;
        match[i] = __ballot(i < per && slot < slots && id[i] == expert);
        mine += __popcll(match[i]);
        const int bound = y - (wave * per + i) * 64;  // slots before y
        if (by_slot && bound > 0) before |= (match[i] & (bound >= 64 ? ~0ull : (1ull << bound) - 1)) != 0;
      }
    });
    if (lane == 0) counts[wave] = mine | before << 16;
    __syncthreads();
    int at = 0, all = 0, seen = 0;
    for (int w = 0; w < WAVES; w++) {
      const int c = counts[w];
      if (w < wave) at += c & 0xffff;
      all += c & 0xffff;
      seen |= c >> 16;
    }
    if (seen) return 0;
    each<0, MOST>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      if (i / 4 * 4 < per) {
        if (match[i] >> lane & 1) list[at + __popcll(match[i] & ((1ull << lane) - 1))] = (uint16_t)((wave * per + i) * 64 + lane);
        at += __popcll(match[i]);
      }
    });
    __syncthreads();
    return all;
  }
};

// A wavefront's sums of rows 16 m ..: to LDS, row r's 16 * NB columns in order from red + r * pitch on
template <bool K1ST, int NB>
__device__ __forceinline__ void put_sums(float *red, int pitch, const f32x4 (&acc)[NB], int lane) {
  const int c = lane & 15, g = lane >> 4;
  each<0, NB>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    const int col = K1ST ? 16 * i + c : NB * c + i;
    each<0, 4>([&](auto rc) __attribute__((always_inline)) { red[(4 * g + rc.value) * pitch + col] = acc[i][rc.value]; });
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
  int64_t pitch_h;     // elements between slots' rows of h
  int64_t plane;       // bf16: bytes between the high parts and the rests
  int slabs;           // of columns of h
  void *h;
  float *row_max, *partial;
  size_t bytes;
};

template <bool BF16>
__device__ __forceinline__ void put_h(const Layout &l, int64_t slot, int col, float h) {
  if constexpr (BF16) {
    uint16_t *at = (uint16_t *)l.h + slot * l.pitch_h + col;
    const float high = __uint_as_float(__float_as_uint(h) & 0xffff0000u);  // cut: rounding may give an infinity, which has no rest
    at[0] = (uint16_t)(__float_as_uint(h) >> 16);
    at[l.plane / 2] = high == h ? 0 : __builtin_bit_cast(uint16_t, (__bf16)(h - high));
  } else
    ((float *)l.h)[slot * l.pitch_h + col] = h;
}

template <int NB>
constexpr int COLS = 16 * NB;

Layout layout_of(const ExpertsParams &p, int h_cols) {
  Layout l;
  const int64_t slots = p.tokens * p.top;
  l.pitch_h = (p.inner + 7) & ~(int64_t)7;
  l.slabs = (int)((p.inner + h_cols - 1) / h_cols);
  const size_t h = (size_t)slots * l.pitch_h * 4, most = ((size_t)slots * l.slabs * 4 + 255) & ~(size_t)255, part = (size_t)slots * p.outputs * 4;
  char *base = (char *)p.workspace;
  l.h = base;
  l.plane = slots * l.pitch_h * 2;
  l.row_max = (float *)(base + ((h + 255) & ~(size_t)255));
  l.partial = (float *)((char *)l.row_max + most);
  l.bytes = ((h + 255) & ~(size_t)255) + most + part;
  return l;
}

// This workgroup's group (of one expert's workgroups) and slabs of columns.  Neighbouring workgroups run on the XCDs in turn; two neighbours in
// the columns should share one, where the cache line between them is: of every 16 workgroups, those of XCD i are shares 2 i and 2 i + 1.
__device__ __forceinline__ void share_of(int slabs, int slabs_each, int &slab, int &last_slab, int &group) {
  int share = blockIdx.x;
  if (share < (int)(gridDim.x & ~15u)) share = (share & ~15) | (share & 7) << 1 | (share >> 3 & 1);
  const int shares = (slabs + slabs_each - 1) / slabs_each;
  group = share / shares;
  slab = (share - group * shares) * slabs_each;
  last_slab = min(slab + slabs_each, slabs);
}

// ---- kernel 1
template <bool BF16, bool I8, bool K1ST, bool GATED, int MT_MOST, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void experts_up_kernel(ExpertsParams p, Layout l, int by_slot, int slabs, int slabs_each) {
  using W = Weights<BF16, I8, K1ST, NB>;
  using R = Rows16<W::OCT>;
  constexpr int HC = GATED ? COLS<NB> / 2 : COLS<NB>, PITCH = COLS<NB> + 4;  // HC: columns of h
  __shared__ uint16_t list[EXPERTS_MAX_SLOTS];
  __shared__ int counts[WAVES];
  __shared__ float red[WAVES * 16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15;
  int slab, last_slab, group;
  share_of(slabs, slabs_each, slab, last_slab, group);
  const int expert = expert_of(p, group, by_slot);
  if ((u32)expert >= (u32)p.experts) return;
  SlotsOf<WAVES> found;
  found.ask(p);
  const int inner = (int)p.inner;
  // (of the groups of columns the first half is the gate's, the other behind it)
  constexpr int GROUPS = COLS<NB> / W::GROUP, GATES = GATED ? GROUPS / 2 : GROUPS;
  struct At {
    int inner, c0;
    __device__ __forceinline__ int operator()(int j) const { return W::column(c0, j % GATES, inner) + (j < GATES ? 0 : inner); }
  };
  Product<BF16, NB, WAVES, W, At> product(p.up, expert, p.hidden, At{inner, 0}, wave, lane);
  product.begin(slab * HC);
  const float *scales = I8 ? p.up.scale + (int64_t)expert * p.up.scale_expert : nullptr;
  const int n = found.find(expert, group, by_slot, list, counts);
  auto rows_from = [&](int r0, auto mt) __attribute__((always_inline)) {
    constexpr int MT = decltype(mt)::value;
    const char *rows[MT];
    const float one[MT] = {};
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = min(r0 + 16 * mc.value + c, n - 1);
      rows[mc.value] = (const char *)p.x + (int64_t)((u32)list[r] / (u32)p.top) * p.ld_x * 2;
    });
    for (int sl = slab; sl < last_slab; sl++) {
      const int tile0 = sl * HC;
      f32x4 acc[MT][NB];
      each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
      product.template rows<R, MT>(acc, rows, 0, one);
      // the next columns' (or rows') weights are on their way while these sums are added
      if (sl + 1 < last_slab) product.begin(tile0 + HC);
      else if (r0 + 16 * MT < n) product.begin(slab * HC);
      each<0, MT>([&](auto mc) __attribute__((always_inline)) {
        constexpr int m = decltype(mc)::value, TPR = 4 * WAVES;  // threads per row
        put_sums<K1ST, NB>(red + wave * 16 * PITCH, PITCH, acc[m], lane);
        __syncthreads();
        const int r = tid / TPR, part = tid % TPR;
        const int slot = r0 + 16 * m + r < n ? list[r0 + 16 * m + r] : -1;
        float most = 0.f;
        for (int j = part; j < HC; j += TPR) {
          // the column that place j holds
          const int col = W::column(tile0, j / W::GROUP, inner) + j % W::GROUP;
          float gate = 0.f, up = 0.f;
          for (int q = 0; q < WAVES; q++) {
            gate += red[(q * 16 + r) * PITCH + j];
            if (GATED) up += red[(q * 16 + r) * PITCH + HC + j];
          }
          if (I8) {
            gate *= scales[col];
            if (GATED) up *= scales[inner + col];
          }
          const float h = GATED ? activate(p.activation, gate) * up : activate(p.activation, gate);
          most = fmaxf(most, fabsf(h));
          if (slot >= 0 && col >= tile0) put_h<BF16>(l, slot, col, h);
        }
        if (slot >= 0 && tile0 + HC >= inner && part < 8 && inner + part < l.pitch_h) put_h<BF16>(l, slot, inner + part, 0.f);
        if (!BF16) {
          for (int d = 1; d < TPR; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
          if (slot >= 0 && part == 0) l.row_max[(int64_t)slot * l.slabs + sl] = most;
        }
        __syncthreads();
      });
    }
  };
  for (int r0 = 0; r0 < n;)
    if (MT_MOST > 2 && n - r0 > 32) rows_from(r0, Int<MT_MOST>{}), r0 += 16 * MT_MOST;
    else if (MT_MOST > 1 && n - r0 > 16) rows_from(r0, Int<2>{}), r0 += 32;
    else rows_from(r0, Int<1>{}), r0 += 16;
}

// ---- kernel 2
template <bool BF16, bool I8, bool K1ST, int MT_MOST, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void experts_down_kernel(ExpertsParams p, Layout l, int by_slot, int slabs, int slabs_each) {
  using W = Weights<BF16, I8, K1ST, NB>;
  using R = RowsOfH<BF16, W::OCT>;
  constexpr int PITCH = COLS<NB> + 4, TPR = 4 * WAVES;  // TPR: threads per row
  __shared__ uint16_t list[EXPERTS_MAX_SLOTS];
  __shared__ int counts[WAVES];
  __shared__ float red[WAVES * 16 * PITCH];
  __shared__ float row_scale[16 * MT_MOST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15;
  int slab, last_slab, group;
  share_of(slabs, slabs_each, slab, last_slab, group);
  const int expert = expert_of(p, group, by_slot);
  if ((u32)expert >= (u32)p.experts) return;
  SlotsOf<WAVES> found;
  found.ask(p);
  const int outputs = (int)p.outputs;
  struct At {
    int outputs, c0;
    __device__ __forceinline__ int operator()(int j) const { return W::column(c0, j, outputs); }
  };
  Product<BF16, NB, WAVES, W, At> product(p.down, expert, p.inner, At{outputs, 0}, wave, lane);
  product.begin(slab * COLS<NB>);
  const float *scales = I8 ? p.down.scale + (int64_t)expert * p.down.scale_expert : nullptr;
  const int n = found.find(expert, group, by_slot, list, counts);
  auto rows_from = [&](int r0, auto mt) __attribute__((always_inline)) {
    constexpr int MT = decltype(mt)::value;
    const char *rows[MT];
    float scale[MT];
    if (!BF16) {  // 2^-e with the row's largest |h| 2^-e in [2^13, 2^14)
      for (int r = tid / TPR; r < 16 * MT; r += 16) {
        float most = 0.f;
        if (r0 + r < n)
          for (int j = tid % TPR; j < l.slabs; j += TPR) most = fmaxf(most, l.row_max[(int64_t)list[r0 + r] * l.slabs + j]);
        for (int d = 1; d < TPR; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        if (tid % TPR == 0) row_scale[r] = fp16_scale(most);
      }
      __syncthreads();
    }
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int r = min(r0 + 16 * mc.value + c, n - 1);
      rows[mc.value] = (const char *)l.h + list[r] * l.pitch_h * (BF16 ? 2 : 4);
      scale[mc.value] = BF16 ? 1.f : row_scale[r - r0];
    });
    float weight[MT];  // of the row that the thread adds up in the end
    each<0, MT>([&](auto mc) __attribute__((always_inline)) {
      const int slot = list[min(r0 + 16 * mc.value + tid / TPR, n - 1)];
      const u32 t = (u32)slot / (u32)p.top;
      weight[mc.value] = p.weights[(int64_t)t * p.ld_weights + (slot - (int)t * p.top)];
    });
    for (int sl = slab; sl < last_slab; sl++) {
      const int tile0 = sl * COLS<NB>;
      f32x4 acc[MT][NB];
      each<0, MT * NB>([&](auto ic) __attribute__((always_inline)) { acc[ic.value / NB][ic.value % NB] = (f32x4){0.f, 0.f, 0.f, 0.f}; });
      product.template rows<R, MT>(acc, rows, l.plane, scale);
      // the next columns' (or rows') weights are on their way while these sums are added
      if (sl + 1 < last_slab) product.begin(tile0 + COLS<NB>);
      else if (r0 + 16 * MT < n) product.begin(slab * COLS<NB>);
      each<0, MT>([&](auto mc) __attribute__((always_inline)) {
        constexpr int m = decltype(mc)::value;
        put_sums<K1ST, NB>(red + wave * 16 * PITCH, PITCH, acc[m], lane);
        __syncthreads();
        const int r = tid / TPR;
        if (r0 + 16 * m + r < n) {
          const int slot = list[r0 + 16 * m + r];
          const float back = BF16 ? 1.f : 1.f / row_scale[16 * m + r];  // (a power of two)
          for (int j = tid % TPR; j < COLS<NB>; j += TPR) {
            const int col = W::column(tile0, j / W::GROUP, outputs) + j % W::GROUP;
            float v = 0.f;
            for (int q = 0; q < WAVES; q++) v += red[(q * 16 + r) * PITCH + j];
            if (!BF16) v *= back;
            if (I8) v *= scales[col];
            l.partial[(int64_t)slot * outputs + col] = v * weight[m];
          }
        }
        __syncthreads();
      });
    }
  };
  for (int r0 = 0; r0 < n;)
    if (MT_MOST > 2 && n - r0 > 32) rows_from(r0, Int<MT_MOST>{}), r0 += 16 * MT_MOST;
    else if (MT_MOST > 1 && n - r0 > 16) rows_from(r0, Int<2>{}), r0 += 32;
    else rows_from(r0, Int<1>{}), r0 += 16;
}

// ---- kernel 3: y[t] = the sum of its slots, eight at a time on their way
template <bool BF16>
__global__ __launch_bounds__(256) void experts_sum_kernel(ExpertsParams p, const float *partial) {
  const int64_t t = blockIdx.y, col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.outputs) return;
  float v = 0.f;
  for (int j0 = 0; j0 < p.top; j0 += 8) {
    float part[8];
    u32 id[8];
    each<0, 8>([&](auto jc) __attribute__((always_inline)) {
      const int j = min(j0 + jc.value, p.top - 1);
      id[jc.value] = (u32)p.ids[t * p.ld_ids + j];
      part[jc.value] = partial[(t * p.top + j) * p.outputs + col];  // (of an id that names no expert: anything)
    });
    each<0, 8>([&](auto jc) __attribute__((always_inline)) {
      if (j0 + jc.value < p.top && id[jc.value] < (u32)p.experts) v += part[jc.value];
    });
  }
  ((uint16_t *)p.out)[t * p.ld_out + col] = BF16 ? tts_gemm_device::f32_to_bf16(v) : tts_gemm_device::f32_to_f16(v);
}


// ---- which variant

// The blocks of 16 columns per workgroup.  Wide tiles read the rows again less often (256 tokens, 64 experts of 4096 x 1536: 559 us of eight blocks of
// contiguous k, 597 of four) and, with contiguous columns, whole cache lines of each row of k (16 experts of int8: 184 us of sixteen, 240 of
// eight); half as wide where that leaves too few workgroups to read at the memory's pace (one token, 8 experts of 2048 x 768: contiguous k 30 us of
// four, 42 of eight; columns 34 of four, 38 of eight, of int8 33 and 51).  Near the borders, layers of 2048 in and out, us wide and half as wide: contiguous
// k, 256 workgroups 44.5 and 43.1, 512 79.7 and 83.2, 1024 142.7 and 138.6, of int8 33.4 and 31.4, 55.6 and 52.5, 97.7 and 89.4; columns, 64 workgroups
// 31.7 and 29.1, 128 36.1 and 35.3, 256 49.2 and 63.1, of int8 40.7 and 32.5, 46.0 and 39.7, 57.3 and 68.5.
// int8 tiles of sixteen blocks with 64 rows at once have more sums than registers (60 to 87 spill).  They are ahead all the same where an expert's rows
// are one turn (128 tokens, 4 of 32 experts of 4096 x 4096: 392 us, 579 of eight), not where they are several (256 tokens, 2 of 8 of 4096 x 2048: 252, 166).
template <bool I8>
int blocks_of(const ExpertMatrix &m, int64_t columns, int groups, int per_block) {
  const int most = m.w_k != 1 && I8 ? 16 : 8;
  return (columns + most * per_block - 1) / (most * per_block) * groups >= (m.w_k == 1 ? 512 : 128) ? most : most / 2;
}

int groups_of(const ExpertsParams &p) { return (int)std::min<int64_t>(p.tokens * p.top, p.experts); }
int down_blocks(const ExpertsParams &p) {
  return p.int8 ? blocks_of<true>(p.down, p.outputs, groups_of(p), 16) : blocks_of<false>(p.down, p.outputs, groups_of(p), 16);
}
int up_blocks(const ExpertsParams &p) {
  const int per_block = p.gated ? 8 : 16;  // columns of h
  return p.int8 ? blocks_of<true>(p.up, p.inner, groups_of(p), per_block) : blocks_of<false>(p.up, p.inner, groups_of(p), per_block);
}
int h_cols(const ExpertsParams &p) { return up_blocks(p) * (p.gated ? 8 : 16); }

// How many slabs of columns a workgroup does one after another: more, while that leaves enough workgroups.  (256 tokens, 6 of 64 experts of 4096 x 1536: 538 us;
// 637 of twice as many slabs, 545 of half as many or one.  32 tokens, 4 of 64 of 2048 x 2048, contiguous columns: 277, 264 and 291, contiguous k 279, 296 and 275.)
int slabs_each(int slabs, int groups) { return (int)std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)slabs * groups / 768)); }
int64_t workgroups_of(int slabs, int groups) {
  const int each = slabs_each(slabs, groups);
  return (int64_t)((slabs + each - 1) / each) * groups;
}

// Rows of an expert at once (in 16s): nearly all of what an expert may have, if tokens pick them alike -- the mean and four times its root -- since
// rows after those read the weights again; but not more, for registers (24 tokens, 16 experts of 2: 16 rows 170 us, 64 rows 195).
int row_blocks(const ExpertsParams &p) {
  const double mean = (double)(p.tokens * p.top) / p.experts, most = std::min<double>((double)p.tokens, mean + 4 * std::sqrt(mean));
  return most <= 16 ? 1 : most <= 32 ? 2 : 4;
}

constexpr int WAVES = 4;

}  // namespace

// The kernels of one type of activations and weights, for up to 32 rows of an expert at once or for more (MANY).  This file is compiled once for
// each of the eight (TTS_EXPERTS_PART: bit 0 bf16, bit 1 int8, bit 2 MANY), side by side, and once for what picks among them.
template <bool BF16, bool I8, bool MANY>
hipError_t launch_experts_as(const ExpertsParams &p, hipStream_t s);

#ifdef TTS_EXPERTS_PART

template <bool BF16, bool I8, bool MANY>
hipError_t launch_experts_as(const ExpertsParams &p, hipStream_t s) {
  const Layout l = layout_of(p, h_cols(p));
  const int groups = groups_of(p), by_slot = groups < p.experts;
  const int nb_up = up_blocks(p), nb_down = down_blocks(p);
  auto up = [&](auto k1st, auto gated, auto mt, auto nb) {
    experts_up_kernel<BF16, I8, decltype(k1st)::value != 0, decltype(gated)::value != 0, decltype(mt)::value, decltype(nb)::value, WAVES>
        <<<dim3((unsigned)workgroups_of(l.slabs, groups)), 64 * WAVES, 0, s>>>(p, l, by_slot, l.slabs, slabs_each(l.slabs, groups));
    return hipGetLastError();
  };
  auto down = [&](auto k1st, auto mt, auto nb) {
    constexpr int width = 16 * decltype(nb)::value;
    const int slabs = (int)((p.outputs + width - 1) / width);
    experts_down_kernel<BF16, I8, decltype(k1st)::value != 0, decltype(mt)::value, decltype(nb)::value, WAVES>
        <<<dim3((unsigned)workgroups_of(slabs, groups)), 64 * WAVES, 0, s>>>(p, l, by_slot, slabs, slabs_each(slabs, groups));
    return hipGetLastError();
  };
  auto with_rows = [&](auto mt) {
    auto up_in = [&](auto gated) {
      if (p.up.w_k != 1) return nb_up == (I8 ? 16 : 8) ? up(Int<0>{}, gated, mt, Int<I8 ? 16 : 8>{}) : up(Int<0>{}, gated, mt, Int<I8 ? 8 : 4>{});
      return nb_up == 8 ? up(Int<1>{}, gated, mt, Int<8>{}) : up(Int<1>{}, gated, mt, Int<4>{});
    };
    const hipError_t e = p.gated ? up_in(Int<1>{}) : up_in(Int<0>{});
    if (e != hipSuccess) return e;
    if (p.down.w_k != 1) return nb_down == (I8 ? 16 : 8) ? down(Int<0>{}, mt, Int<I8 ? 16 : 8>{}) : down(Int<0>{}, mt, Int<I8 ? 8 : 4>{});
    return nb_down == 8 ? down(Int<1>{}, mt, Int<8>{}) : down(Int<1>{}, mt, Int<4>{});
  };
  hipError_t e;
  if constexpr (MANY) e = with_rows(Int<4>{});
  else e = row_blocks(p) == 1 ? with_rows(Int<1>{}) : with_rows(Int<2>{});
  if (e != hipSuccess) return e;
  experts_sum_kernel<BF16><<<dim3((unsigned)((p.outputs + 255) / 256), (unsigned)p.tokens), 256, 0, s>>>(p, l.partial);
  return hipGetLastError();
}

template hipError_t launch_experts_as<(TTS_EXPERTS_PART & 1) != 0, (TTS_EXPERTS_PART & 2) != 0, (TTS_EXPERTS_PART & 4) != 0>(const ExpertsParams &, hipStream_t);

#else

size_t experts_workspace_bytes(const ExpertsParams &p) { return layout_of(p, h_cols(p)).bytes; }

bool experts_fit_a_grid(const ExpertsParams &p) {
  const int down_cols = 16 * down_blocks(p);
  const int64_t most = std::max(workgroups_of((int)((p.inner + h_cols(p) - 1) / h_cols(p)), groups_of(p)), workgroups_of((int)((p.outputs + down_cols - 1) / down_cols), groups_of(p)));
  return most * (64 * WAVES) < (int64_t)1 << 32;
}

hipError_t launch_experts(const ExpertsParams &p, hipStream_t s) {
  auto of = [&](auto many) {
    constexpr bool MANY = decltype(many)::value != 0;
    if (p.bf16) return p.int8 ? launch_experts_as<true, true, MANY>(p, s) : launch_experts_as<true, false, MANY>(p, s);
    return p.int8 ? launch_experts_as<false, true, MANY>(p, s) : launch_experts_as<false, false, MANY>(p, s);
  };
  return row_blocks(p) > 2 ? of(Int<1>{}) : of(Int<0>{});
}

#endif

}  // namespace tts
