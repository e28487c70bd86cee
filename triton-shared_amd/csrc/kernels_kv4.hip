// The paged cache held in 4 bits, written and read.  Of a token's head, for keys and values each:
//   lowest = min(x),  step = (max(x) - min(x)) / 15 in 32 bits, rounded to the type,  code = how many of the borders (n + 1/2) step, n = 0 .. 14, x - lowest is above;
// what it then stands for is code * step + lowest.  A head whose range is not finite in 32 bits (it holds a NaN or an infinity) gets a step of NaN.
// The 16 bits of step and lowest value are the format's: lowest is an element, exactly, and the rounding of step moves what the highest code stands for by 15 / 2 of a step's last place,
// a thirtieth of a step in bf16.
// What bounds them, 16384 tokens of 8 heads of 128: writing 24.9 us, 3.4 TB/s, by some 17 instructions an element (14 to 15 us of issue) behind loads that nothing
// hides, since a lane asks for all it has and then computes; reading 19.7 us, 4.3 TB/s, by memory (at a copy's rate 17 each).  64 tokens: 3.0 and 2.5 us, a launch.
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

// L lanes per head of keys or values; a lane has N times 8 elements, of which neighbouring lanes' are neighbours
template <class T, int L, int N>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4RowsParams p) {
  const Kv4Cache &c = p.cache;
  const int lane = threadIdx.x % L;
  const int item = blockIdx.x * (256 / L) + threadIdx.x / L, t = divided(item, p.by_heads);
  if (t >= p.tokens) return;
  const int rest = item - t * 2 * c.heads, values = rest >= c.heads, head = values ? rest - c.heads : rest;
  const int slot = p.slots[t];
  if (slot < 0 || slot >= c.pages * c.page) return;
  const T *row = (const T *)(values ? p.v : p.k) + (int64_t)t * (values ? p.v_token : p.k_token) + head * (values ? p.v_head : p.k_head);
  row_ops::Dwords<4> x[N];
  for (int n = 0; n < N; n++) {
    const int at = (n * L + lane) * 8;
    x[n] = row_ops::load_dwords<4>((const char *)(row + (at < c.dim ? at : lane * 8 < c.dim ? lane * 8 : 0)));  // (again, where there is nothing)
  }
  auto value = [&](int n, int e) __attribute__((always_inline)) { return (float)from_bits<T>(e & 1 ? x[n].d[e / 2] >> 16 : x[n].d[e / 2]); };
  typedef uint16_t U2 __attribute__((ext_vector_type(2)));
  float low = value(0, 0), high = low;
  U2 most = {0, 0};
  for (int n = 0; n < N; n++)
    for (int e = 0; e < 8; e++) {
      low = fminf(low, value(n, e)), high = fmaxf(high, value(n, e));
      if (e % 2 == 0) most = __builtin_elementwise_max(most, __builtin_bit_cast(U2, x[n].d[e / 2] & 0x7fff7fffu));
    }
  low = over_lanes<L>(low, [](float a, float b) { return fminf(a, b); });
  high = over_lanes<L>(high, [](float a, float b) { return fmaxf(a, b); });
  const uint32_t largest = over_lanes<L>((uint32_t)(most[0] > most[1] ? most[0] : most[1]), [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const float range = high - low;
  const T step_t = (T)(range / 15.f);
  const float step = (float)step_t;
  const bool finite = largest < bits_of((T)__builtin_inff()) && range < __builtin_inff();
  u32 word[N];
  for (int n = 0; n < N; n++) word[n] = 0;
  if (finite && step > 0.f) {
    // The border next to x - lowest, as 32 bits have it, decides between the codes on its sides: that comparison is exact, since borders are whole in 32 bits, but where both
    // are the same there, when what 32 bits leave of the difference decides (seldom: off the way of the others)
    const int power = __builtin_amdgcn_frexp_expf(step);
    const float over = 1.f / __builtin_amdgcn_ldexpf(step, -power);
    for (int n = 0; n < N; n++) {
      float border[8], code[8], nearest = 1.f;
      for (int e = 0; e < 8; e++) {
        const float d = value(n, e) - low;
        border[e] = __builtin_amdgcn_fmed3f(__builtin_rintf(__builtin_fmaf(__builtin_amdgcn_ldexpf(d, -power), over, -0.5f)), 0.f, 14.f);
        const float above = d - (border[e] + 0.5f) * step;
        code[e] = above > 0.f ? border[e] + 1.f : border[e];
        nearest = fminf(nearest, fabsf(above));
      }
      if (__any(nearest == 0.f)) {
        asm volatile("");  // (a branch: not worth computing ahead of it)
        for (int e = 0; e < 8; e++) {
          const float v = value(n, e), d = v - low, back = v - d, left = (v - (d + back)) + (back - low);  // x - lowest is d + left, without an error
          if (d == (border[e] + 0.5f) * step && left > 0.f) code[e] = border[e] + 1.f;
        }
      }
      // (the codes by twos in 32 bits; exact)
      u32 two[4];
      for (int e = 0; e < 4; e++) two[e] = (u32)__builtin_fmaf(code[2 * e + 1], values ? 16.f : 65536.f, code[2 * e]);
      const int apart = values ? 8 : 4;
      word[n] = two[0] | two[1] << apart | two[2] << 2 * apart | two[3] << 3 * apart;
    }
  }
  const Place at = place_of(c, slot, head, values);
  for (int n = 0; n < N; n++)
    if ((n * L + lane) * 8 < c.dim) *(u32 *)(at.codes + (n * L + lane) * 4) = word[n];
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

template <class T, int N>
hipError_t write_n(const Kv4RowsParams &p, hipStream_t s) {
  if (p.cache.dim <= 32) return go<T>(p, 4 / N, s, kv4_write_kernel<T, 4 / N, N>);
  if (p.cache.dim <= 64) return go<T>(p, 8 / N, s, kv4_write_kernel<T, 8 / N, N>);
  if (p.cache.dim <= 128) return go<T>(p, 16 / N, s, kv4_write_kernel<T, 16 / N, N>);
  return go<T>(p, 32 / N, s, kv4_write_kernel<T, 32 / N, N>);
}
// Of many heads a lane takes 32 elements of one, so that what is done once per lane counts less (16384 tokens of 8 heads of 128, side by side: 23.8 us, with 8 elements 30.5); of few
// 8, for a shorter chain (64 tokens: 3.0 us, with 32 elements 4.0; 700: 3.9 and 4.2).
template <class T>
hipError_t write_as(const Kv4RowsParams &p, hipStream_t s) {
  return p.tokens * p.cache.heads > 16384 ? write_n<T, 4>(p, s) : write_n<T, 1>(p, s);
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
