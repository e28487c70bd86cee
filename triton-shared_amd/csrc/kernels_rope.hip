// Norms of queries and keys for each head, and the rotation by position, in one pass over both:
//   y = x * rsqrt(mean(x^2) + eps) * w  (without weights: y = x),  then of the first `rotary` elements pairs (a, b) -> (a cos - b sin, b cos + a sin),
// pair n of them elements n and n + rotary / 2, or 2 n and 2 n + 1, with the cosine and sine of angle n at the row's position.
#include <algorithm>

#include "cache_ops.h"
#include "lanes.h"
#include "row_device.h"
#include "row_ops.h"

namespace tts {

namespace {

// V elements from anywhere, in 32 bits
template <class T, int V>
struct Packed {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Packed<T, V> load(const T *p) {
  Packed<T, V> v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}

// A unit is V pairs: elements lo .. lo + V - 1 and hi .. hi + V - 1 of a head, L lanes per head with N units each, so that a lane has both elements of its
// pairs.  Of neighbouring pairs (INTER) they lie in a row and pair up within it; of the elements behind the rotated ones they are any.
// What bounds it: memory.  8192 tokens of 40 heads of 128 bf16 elements 34 us, 5.0 TB/s, which is what a copy of 1 GiB reaches (cosines, sines and weights come from the caches: they
// are read for every head, 12 bytes of them for 4 of q); one token 2.7 us, a launch and three loads one after another; 617 tokens of 20 heads of 80 (4 pairs a unit) 3.7 us, where units of
// one pair took 7.6.
template <class T, int V, bool INTER, int L, int N>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeParams p) {
  const int heads = p.heads + p.kv_heads, units = p.dim / (2 * V), turned = p.rotary / (2 * V), lane = threadIdx.x % L;
  const int item = blockIdx.x * (256 / L) + threadIdx.x / L;
  const int64_t t = min(divided(item, p.by_all_heads), (int)p.tokens - 1);
  const int head = item - (int)t * heads, position = p.positions[t];
  const bool there = position >= 0 && position < p.places;
  if (head >= heads || (!there && !p.clear)) return;  // (all lanes of a head)
  const float *turn = p.cos_sin + (there ? position : 0) * p.ld_cos_sin;
  int lo[N], hi[N];
  bool mine[N], turns[N];
  Packed<float, V> cos[N], sin[N];
  for (int n = 0; n < N; n++) {
    const int u = lane + n * L, rest = p.rotary + (u - turned) * V;
    mine[n] = u < units, turns[n] = u < turned;
    lo[n] = turns[n] ? (INTER ? 2 * V * u : V * u) : rest;
    hi[n] = turns[n] ? (INTER ? lo[n] + V : lo[n] + p.rotary / 2) : rest + (p.dim - p.rotary) / 2;
    if (turns[n] && there) cos[n] = load<float, V>(turn + V * u), sin[n] = load<float, V>(turn + p.rotary / 2 + V * u);
  }
  const bool q = head < p.heads;
  const int h = q ? head : head - p.heads;
  const T *x = q ? (const T *)p.q + t * p.q_token + h * p.q_head : (const T *)p.k + t * p.k_token + h * p.k_head;
  T *out = q ? (T *)p.q_out + t * p.qo_token + h * p.qo_head : (T *)p.k_out + t * p.ko_token + h * p.ko_head;
  const void *w = q ? p.w_q : p.w_k;
  float a[N][V], b[N][V], squares = 0.f;
  for (int n = 0; n < N; n++) {
    if (!mine[n]) continue;
    const auto va = load<T, V>(x + lo[n]), vb = load<T, V>(x + hi[n]);
    for (int e = 0; e < V; e++) a[n][e] = (float)va.v[e], b[n][e] = (float)vb.v[e], squares += a[n][e] * a[n][e] + b[n][e] * b[n][e];
  }
  if (w) {
    const float r = 1.f / sqrtf(over_lanes<L>(squares, [](float v, float u) { return v + u; }) / (float)p.dim + p.eps);
    for (int n = 0; n < N; n++) {
      if (!mine[n]) continue;
      if (p.w_f32) {
        const auto wa = load<float, V>((const float *)w + lo[n]), wb = load<float, V>((const float *)w + hi[n]);
        for (int e = 0; e < V; e++) a[n][e] = a[n][e] * r * wa.v[e], b[n][e] = b[n][e] * r * wb.v[e];
      } else {
        const auto wa = load<T, V>((const T *)w + lo[n]), wb = load<T, V>((const T *)w + hi[n]);
        for (int e = 0; e < V; e++) a[n][e] = a[n][e] * r * (float)wa.v[e], b[n][e] = b[n][e] * r * (float)wb.v[e];
      }
    }
  }
  for (int n = 0; n < N; n++) {
    if (!mine[n]) continue;
    Packed<T, V> oa, ob;
    if (turns[n] && there) {
      float pair[2 * V];  // the unit's elements in a row
      for (int e = 0; e < V; e++) pair[e] = a[n][e], pair[V + e] = b[n][e];
      for (int e = 0; e < V; e++) {
        float &first = pair[INTER ? 2 * e : e], &second = pair[INTER ? 2 * e + 1 : V + e];
        const float c = cos[n].v[e], s = sin[n].v[e], was = first;
        first = was * c - second * s, second = second * c + was * s;
      }
      for (int e = 0; e < V; e++) a[n][e] = pair[e], b[n][e] = pair[V + e];
    }
    for (int e = 0; e < V; e++) oa.v[e] = (T)(there ? a[n][e] : 0.f), ob.v[e] = (T)(there ? b[n][e] : 0.f);
    __builtin_memcpy(out + lo[n], &oa, sizeof oa);
    __builtin_memcpy(out + hi[n], &ob, sizeof ob);
  }
}

template <class T, int V, bool INTER, int L, int N>
hipError_t go(const RopeParams &p, hipStream_t s) {
  const int64_t heads = p.heads + p.kv_heads, per = 256 / L, each = ((int64_t)1 << 22) * per / heads;  // tokens of a launch (less than 2^32 lanes, and than 2^31 heads)
  for (int64_t at = 0; at < p.tokens; at += each) {
    RopeParams part = p;
    part.by_all_heads = fast_div((uint32_t)heads);
    part.tokens = std::min(each, p.tokens - at);
    part.positions += at;
    part.q = (const T *)p.q + at * p.q_token, part.k = (const T *)p.k + at * p.k_token;
    part.q_out = (T *)p.q_out + at * p.qo_token, part.k_out = (T *)p.k_out + at * p.ko_token;
    qk_norm_rope_kernel<T, V, INTER, L, N><<<dim3((unsigned)((part.tokens * heads + per - 1) / per)), 256, 0, s>>>(part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Units of 8 pairs where what is rotated and what is not are whole ones, of 4, or of one.
template <class T, bool INTER>
hipError_t launch_of(const RopeParams &p, hipStream_t s) {
  if (p.rotary % 16 == 0 && p.dim % 16 == 0) {
    const int units = p.dim / 16;
    if (units <= 4) return go<T, 8, INTER, 4, 1>(p, s);
    if (units <= 8) return go<T, 8, INTER, 8, 1>(p, s);
    if (units <= 16) return go<T, 8, INTER, 16, 1>(p, s);
    return go<T, 8, INTER, 32, 1>(p, s);
  }
  if (p.rotary % 8 == 0 && p.dim % 8 == 0) return p.dim <= 128 ? go<T, 4, INTER, 16, 1>(p, s) : go<T, 4, INTER, 64, 1>(p, s);
  return go<T, 1, INTER, 64, ROPE_MAX_DIM / 128>(p, s);
}

template <class T>
hipError_t launch_as(const RopeParams &p, hipStream_t s) {
  return p.interleaved ? launch_of<T, true>(p, s) : launch_of<T, false>(p, s);
}

}  // namespace

hipError_t launch_rope(const RopeParams &p, hipStream_t s) {
  return p.elem == ELEM_F32 ? launch_as<float>(p, s) : p.elem == ELEM_F16 ? launch_as<_Float16>(p, s) : launch_as<__bf16>(p, s);
}

}  // namespace tts
