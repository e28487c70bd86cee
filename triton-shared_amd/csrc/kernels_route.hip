// The router of a mixture-of-experts layer.  Per token, from its logits l over the experts:
//   s = softmax(l) or sigmoid(l);  c = s + bias, or l itself without a bias (the same order, and no two logits that differ
//   become equal);  the `top` largest c, ties to the lowest expert;  weight = scale * s / (the sum of the chosen s).
// A logit of -inf (a masked expert), a c of -inf and a NaN are never chosen; where fewer than `top` are left the rest of the row is expert -1
// of weight 0.  A row that holds a NaN has NaN for its chosen experts' weights, as the formula gives, and so has the softmax of one that holds +inf.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kernels.h"
#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

// v of the lane N after, around 16 lanes
template <int N, class T>
__device__ __forceinline__ T rotated(T v) {
  constexpr int DW = sizeof(T) / 4;
  int d[DW];
  __builtin_memcpy(d, &v, sizeof v);
  for (int i = 0; i < DW; i++) d[i] = __builtin_amdgcn_update_dpp(d[i], d[i], 0x120 + N, 0xf, 0xf, false);  // row_ror
  __builtin_memcpy(&v, d, sizeof v);
  return v;
}

// f over G neighbouring lanes' values, in all of them: within 16 lanes by DPP moves: a choice's chain of reductions waits for each (one token of
// 128 experts 8.2 us with moves through LDS, 4.7 so)
template <int G, class T, class F>
__device__ __forceinline__ T over_lanes(T v, F f) {
  v = f(v, rotated<8>(v));
  v = f(v, rotated<4>(v));
  v = f(v, rotated<2>(v));
  v = f(v, rotated<1>(v));
  for (int d = 16; d < G; d *= 2) v = f(v, __shfl_xor(v, d));
  return v;
}

template <class T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<_Float16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float widen<__bf16>(__bf16 v) { return (float)v; }

// The `top` largest of G lanes' c, in turn: lane n % G keeps the n'th expert in chosen[n / G].  `close`, where it is given: whether one of them, or the first that is left, is less than `apart` from the one before, and more than its rounding;  `least`: what
// no c that belongs among them is below, off by as much.
template <class C, int G, int N>
__device__ __forceinline__ void choose(const C (&c)[N], int lane, int top, int (&chosen)[ROUTE_MAX_TOP / G], float apart, bool *close, float *least) {
  unsigned taken = 0;
  C before = INFINITY;
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) chosen[h] = -1;
  for (int n = 0; n < top + (close ? 1 : 0); n++) {
    C best = -INFINITY;
    int at = -1;
    for (int j = 0; j < N; j++)
      if (!(taken >> j & 1) && c[j] > best) best = c[j], at = j;
    const C winner = over_lanes<G>(best, [](C a, C b) { return a > b ? a : b; });
    const int mine = best == winner && at >= 0 ? at * G + lane : INT_MAX;
    const int expert = over_lanes<G>(mine, [](int a, int b) { return a < b ? a : b; });
    const bool any = expert != INT_MAX;
    if (any && expert == mine) taken |= 1u << at;
    if (close && any) {
      const float enough = apart + 0x1p-23f * fabsf((float)winner);  // (c's own rounding)
      *close |= !((float)(before - winner) > enough);
      if (n < top) *least = (float)winner - enough;
    }
    before = winner;
    for (int h = 0; h < ROUTE_MAX_TOP / G; h++)
      if (n < top && n == h * G + lane) chosen[h] = any ? expert : -1;
  }
}

template <int N>
__device__ __forceinline__ float pick(const float (&v)[N], int j) {
  float r = v[0];
  row_ops::each<1, N>([&](auto ic) __attribute__((always_inline)) { r = ic.value == j ? v[ic.value] : r; });  // (indexed by constants: in registers)
  return r;
}

__device__ __forceinline__ float sigmoid(float l) {
  const float x = expf(-fabsf(l));
  return (l < 0.f ? x : 1.f) / (1.f + x);
}

// The logarithm under which a score is 0 (64 bits hold none there): experts that a mask of the type's lowest value leaves have no weight.
constexpr float NO_SCORE = -745.f;

// G lanes per token; lane i of them holds experts i, i + G, ... (N of them).  Which expert is chosen shows whole, so where scores get a bias
// the choice is that of c in 64 bits: 32 bits decide it unless two that matter are near each other, which is seldom (a token in a thousand of
// the one measured); then the candidates' c is computed in 64 bits and the choice made again.
// What bounds it: one token 4.5 us, a launch and a chain of two reductions per choice; 16384 tokens of 256 fp32 logits 11 us without a bias (17 MB, 3.3
// at a copy's rate: a choice is some 160 instructions of four tokens' lanes), 21 with one, of which the last wavefront's second choice is
// half: it starts on code that is not in the instruction cache yet.
template <class T, bool BIAS, int G, int N>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteParams p) {
  const int64_t token = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const bool live = token < p.tokens;  // (lanes of no token go along: the reductions are over whole groups)
  const T *row = (const T *)p.logits + (live ? token : 0) * p.ld;
  float l[N], bias[N];
  if constexpr (BIAS)
    for (int j = 0; j < N; j++) bias[j] = p.bias[min(j * G + lane, p.experts - 1)];  // (all on their way, with the logits)
  bool nan = false;
  float most = -INFINITY;
  for (int j = 0; j < N; j++) {
    const int e = j * G + lane;
    const float v = widen<T>(row[min(e, p.experts - 1)]);
    l[j] = e < p.experts ? v : -INFINITY;
    nan |= l[j] != l[j];
    most = fmaxf(most, l[j]);
  }
  most = over_lanes<G>(most, [](float a, float b) { return fmaxf(a, b); });
  nan = over_lanes<G>((int)nan, [](int a, int b) { return a | b; });
  if (!p.sigmoid && most == INFINITY) {  // the softmax is NaN, and what is chosen is told by its limit: infinite logits share it, nothing is left for others
    nan = true;
    if constexpr (BIAS) {
      for (int j = 0; j < N; j++) l[j] = l[j] == INFINITY ? 0.f : l[j] > -INFINITY ? -FLT_MAX : l[j];
      most = 0.f;
    }
  }
  int chosen[ROUTE_MAX_TOP / G];
  float held[ROUTE_MAX_TOP / G], sum = 0.f;
  const auto add = [](auto a, auto b) { return a + b; };
  if (!p.sigmoid && (BIAS || !p.renormalize)) {  // the softmax's sum, where the chosen ones' shares of it are asked for
    for (int j = 0; j < N; j++)
      if (l[j] > -INFINITY) sum += expf(l[j] - most);
    sum = over_lanes<G>(sum, add);
  }
  if constexpr (BIAS) {
    float c[N];
    for (int j = 0; j < N; j++) {
      const float score = p.sigmoid ? sigmoid(l[j]) : expf(l[j] - most) / sum;
      c[j] = l[j] > -INFINITY ? score + bias[j] : -INFINITY;  // (experts that are not there have logits of -inf)
    }
    // Scores are off by less than half of `apart`.  sigmoid: an exponential, a sum and a quotient, 2^-21.6 of the score in all; softmax: the sum of up to
    // 1024 exponentials besides, 22 roundings, and 2^-24 of an argument x, x e^-x < 1
    bool close = false;
    float least = -INFINITY;
    choose<float, G, N>(c, lane, p.top, chosen, p.sigmoid ? 0x1p-20f : 0x1p-17f, &close, &least);
    if (close) {
      double whole = 0.0, exact[N];
      if (!p.sigmoid) {
#pragma unroll 1
        for (int j = 0; j < N; j++) {
          const float lj = pick<N>(l, j);
          if (lj > -INFINITY) whole += exp((double)lj - (double)most);
        }
        whole = over_lanes<G>(whole, add);
      }
      unsigned near = 0;  // the experts that may belong among the chosen
      row_ops::each<0, N>([&](auto jc) __attribute__((always_inline)) {
        exact[jc.value] = -INFINITY;
        near |= (unsigned)(c[jc.value] > -INFINITY && !(c[jc.value] < least)) << jc.value;
      });
#pragma unroll 1
      while (near) {
        const int j = __builtin_ctz(near);
        near &= near - 1;
        const float lj = pick<N>(l, j);
        // sigmoid(l) = x / (1 + x) with x = exp(l), or 1 / (1 + exp(-l)) where that is the smaller
        const double x = exp(p.sigmoid ? -fabs((double)lj) : (double)lj - (double)most);
        const double v = (p.sigmoid ? (lj < 0.f ? x : 1.0) / (1.0 + x) : x / whole) + (double)pick<N>(bias, j);
        row_ops::each<0, N>([&](auto ic) __attribute__((always_inline)) { exact[ic.value] = ic.value == j ? v : exact[ic.value]; });
      }
      choose<double, G, N>(exact, lane, p.top, chosen, 0.f, nullptr, nullptr);
    }
  } else
    choose<float, G, N>(l, lane, p.top, chosen, 0.f, nullptr, nullptr);
  // the scores of the chosen ones, all at once
  float z[ROUTE_MAX_TOP / G], total = 0.f;
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) z[h] = chosen[h] >= 0 ? widen<T>(row[chosen[h]]) : -INFINITY;
  auto hold = [&](auto score) __attribute__((always_inline)) {
    total = 0.f;
    for (int h = 0; h < ROUTE_MAX_TOP / G; h++) {
      float s = 0.f;
      if (chosen[h] >= 0) s = nan ? NAN : score(z[h]);
      held[h] = s;
      total += s;
    }
    total = over_lanes<G>(total, add);
  };
  hold([&](float z) __attribute__((always_inline)) {
    if (p.sigmoid) return sigmoid(z);
    const float s = expf(z - most);
    return p.renormalize ? s : s / sum;
  });
  if (p.renormalize && total < 0.5f) {
    // Some may be below what 32 bits hold, and not small in the sum of them: again without the factor that takes them all there, which
    // divides out.  exp(z) is exp(z - largest), and where all are negative sigmoid(z) = exp(z) / (1 + exp(z)) is exp(z - largest) / (1 + exp(z)).
    // (In every row instead: 21.8 us of the 16384 tokens below instead of 21.6.)
    float largest = z[0];
    for (int h = 1; h < ROUTE_MAX_TOP / G; h++) largest = fmaxf(largest, z[h]);
    largest = over_lanes<G>(largest, [](float a, float b) { return fmaxf(a, b); });
    hold([&](float z) __attribute__((always_inline)) {
      if (z - (p.sigmoid ? 0.f : most) < NO_SCORE) return 0.f;
      if (p.sigmoid) return largest < 0.f ? expf(z - largest) / (1.f + expf(z)) : sigmoid(z);
      return expf(z - largest);
    });
  }
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) {
    const int n = h * G + lane;
    if (live && n < p.top) {
      p.ids[token * p.ld_ids + n] = chosen[h];
      p.weights[token * p.ld_weights + n] = held[h] == 0.f ? 0.f : held[h] / (p.renormalize ? total : 1.f) * p.scale;
    }
  }
}

template <class T, bool BIAS>
hipError_t launch_as(const RouteParams &p, hipStream_t s) {
  // a launch has less than 2^32 lanes in all (the runtime starts the rest of them without an error): more tokens go one part after another
  auto go = [&](auto kernel, int lanes) {
    const int64_t each = ((int64_t)1 << 31) / lanes;
    for (int64_t at = 0; at < p.tokens; at += each) {
      RouteParams part = p;
      part.tokens = std::min(each, p.tokens - at);
      part.logits = (const T *)p.logits + at * p.ld, part.ids += at * p.ld_ids, part.weights += at * p.ld_weights;
      kernel<<<dim3((unsigned)((part.tokens + 256 / lanes - 1) / (256 / lanes))), 256, 0, s>>>(part);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (p.experts <= 64) return go(moe_route_kernel<T, BIAS, 16, 4>, 16);
  if (p.experts <= 128) return go(moe_route_kernel<T, BIAS, 16, 8>, 16);
  if (p.experts <= 256) return go(moe_route_kernel<T, BIAS, 16, 16>, 16);
  if (p.experts <= 512) return go(moe_route_kernel<T, BIAS, 64, 8>, 64);
  return go(moe_route_kernel<T, BIAS, 64, 16>, 64);
}

template <class T>
hipError_t launch_of(const RouteParams &p, hipStream_t s) {
  return p.bias ? launch_as<T, true>(p, s) : launch_as<T, false>(p, s);
}

}  // namespace

hipError_t launch_route(const RouteParams &p, hipStream_t s) {
  return p.elem == ELEM_F32 ? launch_of<float>(p, s) : p.elem == ELEM_F16 ? launch_of<_Float16>(p, s) : launch_of<__bf16>(p, s);
}

}  // namespace tts
