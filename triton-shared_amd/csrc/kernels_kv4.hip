// The paged cache held in 4 bits, written and read.  Of a token's head, for keys and values each:
//   lowest = min(x),  step = (max(x) - min(x)) / 15 in 32 bits, rounded to the type,  code = how many of the borders (n + 1/2) step, n = 0 .. 14, x - lowest is above;
// what it then stands for is code * step + lowest.  A head whose range is not finite in 32 bits (it holds a NaN or an infinity) gets a step of NaN.
#include <algorithm>

#include "cache_ops.h"
#include "lanes.h"
#include "row_device.h"

namespace tts {

namespace {

using row_ops::u32;

template <class T>
__device__ __forceinline__ u32 bits_of(T v) { return (u32)__builtin_bit_cast(uint16_t, v); }
template <class T>
__device__ __forceinline__ T from_bits(u32 v) { return __builtin_bit_cast(T, (uint16_t)v); }

struct Place {
  char *codes, *pair;
};
// where a slot's head is (`values`: its value, else its key)
__device__ __forceinline__ Place place_of(const Kv4Cache &c, int slot, int head, int values) {
  const int page = divided(slot, c.by_page), at = slot - page * c.page;
  char *base = (char *)c.base + page * c.page_bytes + head * c.head_bytes;
  return {base + ((int64_t)values * c.page + at) * (c.dim / 2), base + (int64_t)c.page * c.dim + ((int64_t)values * c.page + at) * 4};
}

// which bits of a word hold element e
__device__ __forceinline__ constexpr int shift_of(int e, bool values) { return values ? 4 * e : (e & 1) * 16 + (e / 2) * 4; }

// L lanes per head of keys or values, 8 elements a lane
template <class T, int L>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4RowsParams p) {
  const Kv4Cache &c = p.cache;
  const int lane = threadIdx.x % L;
  const int item = blockIdx.x * (256 / L) + threadIdx.x / L, t = divided(item, p.by_heads);
  if (t >= p.tokens) return;
  const int rest = item - t * 2 * c.heads, values = rest >= c.heads, head = values ? rest - c.heads : rest;
  const int slot = p.slots[t];
  if (slot < 0 || slot >= c.pages * c.page) return;
  const bool mine = lane * 8 < c.dim;
  const T *row = (const T *)(values ? p.v : p.k) + (int64_t)t * (values ? p.v_token : p.k_token) + head * (values ? p.v_head : p.k_head);
  T x[8];
  __builtin_memcpy(x, row + (mine ? lane * 8 : 0), sizeof x);
  float low = (float)x[0], high = low;
  int finite = 1;
  for (int e = 0; e < 8; e++) {
    const float v = (float)x[e];
    low = fminf(low, v), high = fmaxf(high, v);
    finite &= __builtin_fabsf(v) < __builtin_inff();
  }
  low = over_lanes<L>(low, [](float a, float b) { return fminf(a, b); });
  high = over_lanes<L>(high, [](float a, float b) { return fmaxf(a, b); });
  finite = over_lanes<L>(finite, [](int a, int b) { return a & b; });
  const float range = high - low;
  const T step_t = (T)(range / 15.f);
  const float step = (float)step_t;
  finite &= range < __builtin_inff();
  u32 word = 0;
  if (finite && step > 0.f) {
    // The border next to x - lowest, as 32 bits have it, decides between the codes on its sides: that comparison is exact, since borders are whole in 32 bits, but where both
    // are the same there, when what 32 bits leave of the difference decides (seldom: off the way of the others)
    const int power = __builtin_amdgcn_frexp_expf(step);
    const float over = 1.f / __builtin_amdgcn_ldexpf(step, -power);
    float d[8], border[8], code[8];
    bool even = false;
    for (int e = 0; e < 8; e++) {
      d[e] = (float)x[e] - low;
      border[e] = __builtin_amdgcn_fmed3f(__builtin_rintf(__builtin_fmaf(__builtin_amdgcn_ldexpf(d[e], -power), over, -0.5f)), 0.f, 14.f);
      const float at = (border[e] + 0.5f) * step;
      code[e] = d[e] > at ? border[e] + 1.f : border[e];
      even |= d[e] == at;
    }
    if (__any(even))
      for (int e = 0; e < 8; e++) {
        const float v = (float)x[e], back = v - d[e], rest = (v - (d[e] + back)) + (back - low);  // x - lowest is d + rest, without an error
        if (d[e] == (border[e] + 0.5f) * step && rest > 0.f) code[e] = border[e] + 1.f;
      }
    // (the codes by twos in 32 bits; exact)
    u32 two[4];
    for (int e = 0; e < 4; e++) two[e] = (u32)__builtin_fmaf(code[2 * e + 1], values ? 16.f : 65536.f, code[2 * e]);
    word = values ? two[0] | two[1] << 8 | two[2] << 16 | two[3] << 24 : two[0] | two[1] << 4 | two[2] << 8 | two[3] << 12;
  }
  const Place at = place_of(c, slot, head, values);
  if (mine) *(u32 *)(at.codes + lane * 4) = word;
  if (lane == 0) *(u32 *)at.pair = finite ? bits_of(step_t) | bits_of((T)(low + 0.f)) << 16 : bits_of((T)__builtin_nanf(""));
}

// (a token without a slot: zeros)
template <class T, int L>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowsParams p) {
  const Kv4Cache &c = p.cache;
  const int lane = threadIdx.x % L;
  const int item = blockIdx.x * (256 / L) + threadIdx.x / L, t = divided(item, p.by_heads);
  if (t >= p.tokens || lane * 8 >= c.dim) return;
  const int rest = item - t * 2 * c.heads, values = rest >= c.heads, head = values ? rest - c.heads : rest;
  const int slot = p.slots[t];
  T *row = (T *)(values ? p.v : p.k) + (int64_t)t * (values ? p.v_token : p.k_token) + head * (values ? p.v_head : p.k_head);
  T x[8] = {};
  if (slot >= 0 && slot < c.pages * c.page) {
    const Place at = place_of(c, slot, head, values);
    const u32 word = *(const u32 *)(at.codes + lane * 4), pair = *(const u32 *)at.pair;
    const float step = (float)from_bits<T>(pair), low = (float)from_bits<T>(pair >> 16);
    for (int e = 0; e < 8; e++) x[e] = (T)((float)(word >> (values ? shift_of(e, true) : shift_of(e, false)) & 15) * step + low);
  }
  __builtin_memcpy(row + lane * 8, x, sizeof x);
}

template <class T, class K>
hipError_t go(const Kv4RowsParams &p, int lanes, hipStream_t s, K kernel) {
  const int64_t per = 256 / lanes, heads = 2 * p.cache.heads, each = ((int64_t)1 << 22) * per / heads;  // tokens of a launch (less than 2^32 lanes, and than 2^31 heads)
  for (int64_t at = 0; at < p.tokens; at += each) {
    Kv4RowsParams part = p;
    part.by_heads = fast_div((uint32_t)heads);
    part.tokens = std::min(each, p.tokens - at);
    part.slots += at;
    part.k = (T *)p.k + at * p.k_token, part.v = (T *)p.v + at * p.v_token;
    kernel<<<dim3((unsigned)((part.tokens * heads + per - 1) / per)), 256, 0, s>>>(part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T>
hipError_t write_as(const Kv4RowsParams &p, hipStream_t s) {
  if (p.cache.dim <= 32) return go<T>(p, 4, s, kv4_write_kernel<T, 4>);
  if (p.cache.dim <= 64) return go<T>(p, 8, s, kv4_write_kernel<T, 8>);
  if (p.cache.dim <= 128) return go<T>(p, 16, s, kv4_write_kernel<T, 16>);
  return go<T>(p, 32, s, kv4_write_kernel<T, 32>);
}
template <class T>
hipError_t read_as(const Kv4RowsParams &p, hipStream_t s) {
  if (p.cache.dim <= 32) return go<T>(p, 4, s, kv4_read_kernel<T, 4>);
  if (p.cache.dim <= 64) return go<T>(p, 8, s, kv4_read_kernel<T, 8>);
  if (p.cache.dim <= 128) return go<T>(p, 16, s, kv4_read_kernel<T, 16>);
  return go<T>(p, 32, s, kv4_read_kernel<T, 32>);
}

}  // namespace

hipError_t launch_kv4_write(const Kv4RowsParams &p, hipStream_t s) { return p.cache.bf16 ? write_as<__bf16>(p, s) : write_as<_Float16>(p, s); }
hipError_t launch_kv4_read(const Kv4RowsParams &p, hipStream_t s) { return p.cache.bf16 ? read_as<__bf16>(p, s) : read_as<_Float16>(p, s); }

}  // namespace tts
