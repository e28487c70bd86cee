// The router of a mixture-of-experts layer.  Per token, from its logits l over the experts:
//   s = softmax(l) or sigmoid(l);  c = s + bias, or l itself without a bias (the same order, and no two logits that differ
//   become equal);  the `top` largest c, ties to the lowest expert;  weight = scale * s / (the sum of the chosen s).
// A logit of -inf (a masked expert), a c of -inf and a NaN are never chosen; where fewer than `top` are left the rest of the row is expert -1
// of weight 0.  A row that holds a NaN has NaN for its chosen experts' weights, as the formula gives.
#include <cmath>

#include "kernels.h"
#include "row_ops.h"

namespace tts {

namespace {

// the largest of G neighbouring lanes' values, in all of them
template <int G, class T, class F>
__device__ __forceinline__ T over_lanes(T v, F f) {
  for (int d = 1; d < G; d *= 2) v = f(v, __shfl_xor(v, d));
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

// G lanes per token; lane i of them holds experts i, i + G, ... (N of them).  C: the type that c is compared in.  Scores that get
// a bias are computed in 64 bits: rounded to 32, scores that differ by less than 2^-24 would tie, and which expert is chosen shows whole.
template <class T, class C, int G, int N>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteParams p) {
  const int64_t token = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const bool live = token < p.tokens;  // (lanes of no token go along: the reductions are over whole groups)
  const T *row = (const T *)p.logits + (live ? token : 0) * p.ld;
  constexpr bool BIAS = sizeof(C) == 8;
  float l[N];
  bool nan = false;
  float most = -INFINITY;
  for (int j = 0; j < N; j++) {
    const int e = j * G + lane;
    l[j] = e < p.experts ? widen<T>(row[e]) : -INFINITY;
    nan |= l[j] != l[j];
    most = fmaxf(most, l[j]);
  }
  most = over_lanes<G>(most, [](float a, float b) { return fmaxf(a, b); });
  nan = over_lanes<G>((int)nan, [](int a, int b) { return a | b; });
  // the softmax's sum, where the chosen ones' shares of it are asked for
  C sum = 0;
  if (!p.sigmoid && (BIAS || !p.renormalize)) {
    for (int j = 0; j < N; j++)
      if (l[j] > -INFINITY) sum += exp((C)l[j] - (C)most);
    sum = over_lanes<G>(sum, [](C a, C b) { return a + b; });
  }
  C c[N];
  for (int j = 0; j < N; j++) {
    const int e = j * G + lane;
    c[j] = (C)l[j];
    if constexpr (BIAS) {
      if (e < p.experts && l[j] > -INFINITY) c[j] = (p.sigmoid ? 1.0 / (1.0 + exp(-(double)l[j])) : exp((double)l[j] - (double)most) / sum) + (double)p.bias[e];
      else c[j] = -INFINITY;
    }
  }
  unsigned taken = 0;
  float total = 0.f, held[ROUTE_MAX_TOP / G];  // lane i holds choices i, i + G, ...
  int chosen[ROUTE_MAX_TOP / G];
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) held[h] = 0.f, chosen[h] = -1;
  for (int n = 0; n < p.top; n++) {
    C best = -INFINITY;
    int at = -1;
    float logit = 0.f;
    for (int j = 0; j < N; j++)
      if (!(taken >> j & 1) && c[j] > best) best = c[j], at = j, logit = l[j];
    const C winner = over_lanes<G>(best, [](C a, C b) { return a > b ? a : b; });
    const int mine = best == winner && at >= 0 ? at * G + lane : INT_MAX;
    const int expert = over_lanes<G>(mine, [](int a, int b) { return a < b ? a : b; });
    const bool any = expert != INT_MAX;
    if (any && expert == mine) taken |= 1u << at;
    const float z = __shfl(logit, any ? expert % G : 0, G);  // the chosen one's logit
    for (int h = 0; h < ROUTE_MAX_TOP / G; h++)
      if (n == h * G + lane) held[h] = z, chosen[h] = any ? expert : -1;
  }
  // the scores of the chosen ones, all at once
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) {
    const float z = held[h];
    float s = 0.f;
    if (chosen[h] >= 0) {
      s = p.sigmoid ? (float)(1.0 / (1.0 + exp(-(double)z))) : expf(z - most);
      if (!p.sigmoid && !p.renormalize) s = (float)((C)s / sum);
      if (nan) s = NAN;
    }
    held[h] = s;
    total += s;
  }
  total = over_lanes<G>(total, [](float a, float b) { return a + b; });
  for (int h = 0; h < ROUTE_MAX_TOP / G; h++) {
    const int n = h * G + lane;
    if (live && n < p.top) {
      p.ids[token * p.ld_ids + n] = chosen[h];
      p.weights[token * p.ld_weights + n] = held[h] == 0.f ? 0.f : held[h] / (p.renormalize ? total : 1.f) * p.scale;
    }
  }
}

template <class T, class C>
hipError_t launch_as(const RouteParams &p, hipStream_t s) {
  auto go = [&](auto kernel, int lanes) {
    kernel<<<dim3((unsigned)((p.tokens + 256 / lanes - 1) / (256 / lanes))), 256, 0, s>>>(p);
    return hipGetLastError();
  };
  if (p.experts <= 64) return go(moe_route_kernel<T, C, 16, 4>, 16);
  if (p.experts <= 128) return go(moe_route_kernel<T, C, 16, 8>, 16);
  if (p.experts <= 256) return go(moe_route_kernel<T, C, 16, 16>, 16);
  if (p.experts <= 512) return go(moe_route_kernel<T, C, 64, 8>, 64);
  return go(moe_route_kernel<T, C, 64, 16>, 64);
}

template <class T>
hipError_t launch_of(const RouteParams &p, hipStream_t s) {
  return p.bias ? launch_as<T, double>(p, s) : launch_as<T, float>(p, s);
}

}  // namespace

hipError_t launch_route(const RouteParams &p, hipStream_t s) {
  return p.elem == ELEM_F32 ? launch_of<float>(p, s) : p.elem == ELEM_F16 ? launch_of<_Float16>(p, s) : launch_of<__bf16>(p, s);
}

}  // namespace tts
