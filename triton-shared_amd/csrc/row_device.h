// Device code shared by the operators whose weights are picked per row (kernels_experts.hip, kernels_lora.hip).
#pragma once
#include "gemm_device.h"

namespace tts {
namespace row_ops {

using tts_gemm_device::bf16x8;
using tts_gemm_device::f16x2;
using tts_gemm_device::f16x8;
using tts_gemm_device::f32x4;

typedef uint32_t u32;

template <int I>
struct Int {
  static constexpr int value = I;
};
template <int B, int E, class F>
__device__ __forceinline__ void each(F &&f) {
  if constexpr (B < E) {
    f(Int<B>{});
    each<B + 1, E>(f);
  }
}

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// DW dwords from any element's address
template <int DW>
struct Dwords {
  u32 d[DW];
};
template <int DW>
__device__ __forceinline__ Dwords<DW> load_dwords(const char *p) {
  Dwords<DW> v;
  __builtin_memcpy(&v, p, 4 * DW);
  return v;
}

// the same for what is read once: it leaves the caches to what is read again
template <int DW>
__device__ __forceinline__ Dwords<DW> stream_dwords(const char *p) {
  if constexpr (DW == 1) {
    typedef u32 U1 __attribute__((aligned(1)));
    return {__builtin_nontemporal_load((const U1 *)p)};
  } else {
    typedef u32 V __attribute__((ext_vector_type(DW)));
    typedef V Unaligned __attribute__((aligned(1)));
    return __builtin_bit_cast(Dwords<DW>, (V)__builtin_nontemporal_load((const Unaligned *)p));
  }
}

// the first `valid` of 16 bytes, zeros behind: by a load that ends with them (the row they end has at least 16 bytes)
__device__ __forceinline__ Dwords<4> load_part(const char *p, int valid) {
  if (valid <= 0) return Dwords<4>{};
  const int back = valid < 16 ? 16 - valid : 0;
  Dwords<4> v = load_dwords<4>(p - back);
  if (back & 8) v = {v.d[2], v.d[3], 0, 0};
  if (back & 4) v = {v.d[1], v.d[2], v.d[3], 0};
  const u32 next[4] = {v.d[1], v.d[2], v.d[3], 0};
  each<0, 4>([&](auto ic) __attribute__((always_inline)) { v.d[ic.value] = __builtin_amdgcn_alignbyte(next[ic.value], v.d[ic.value], back & 3); });
  return v;
}

// two int8 weights, in bytes 0 and 2 of `v` (the others zero), as a pair of 16-bit floats: exact
template <bool BF16>
__device__ __forceinline__ u32 widen_pair(u32 v) {
  if constexpr (BF16) {
    const float lo = (float)(int8_t)v, hi = (float)(int8_t)(v >> 16);
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
  }
  // with its sign flipped a byte is b + 128, and behind 0x64 in the high byte the fp16 1024 + b + 128
  const f16x2 biased = __builtin_bit_cast(f16x2, v ^ 0x64806480u), off = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(u32, biased - off);
}

// Eight values of fp32, times a power of two, as the sum of two operands of eight 16-bit values: PART 0 the high part, PART 1 the
// rest of them.  bf16: the high half, cut (rounding may give an infinity), and the rest rounded.  An infinity has no rest.
template <bool BF16, int PART>
__device__ __forceinline__ uint4 split_part(const float (&v)[8], float scale) {
  u32 w[4];
  each<0, 4>([&](auto pc) __attribute__((always_inline)) {
    constexpr int p = decltype(pc)::value;
    if constexpr (BF16) {
      const u32 a = __float_as_uint(v[2 * p]), b = __float_as_uint(v[2 * p + 1]);
      if constexpr (PART == 0) w[p] = __builtin_amdgcn_perm(b, a, 0x07060302);
      else {
        const float ha = __uint_as_float(a & 0xffff0000u), hb = __uint_as_float(b & 0xffff0000u);
        const float ra = ha == v[2 * p] ? 0.f : v[2 * p] - ha, rb = hb == v[2 * p + 1] ? 0.f : v[2 * p + 1] - hb;
        w[p] = (u32)__builtin_bit_cast(uint16_t, (__bf16)ra) | (u32)__builtin_bit_cast(uint16_t, (__bf16)rb) << 16;
      }
    } else {
      const float a = v[2 * p] * scale, b = v[2 * p + 1] * scale;
      const auto high = __builtin_amdgcn_cvt_pkrtz(a, b);
      if constexpr (PART == 0) w[p] = __builtin_bit_cast(u32, high);
      else {
        const float ha = (float)high[0], hb = (float)high[1];
        w[p] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(ha == a ? 0.f : a - ha, hb == b ? 0.f : b - hb));
      }
    }
  });
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// the power of two that takes a row whose largest magnitude is `most` below 2^14, where fp16 holds it in full (1 if that is 0, inf or NaN)
__device__ __forceinline__ float fp16_scale(float most) {
  if (!(most > 0.f && most < __builtin_inff())) return 1.f;
  return __builtin_amdgcn_ldexpf(1.f, max(-126, min(126, 14 - __builtin_amdgcn_frexp_expf(most))));
}

}  // namespace row_ops
}  // namespace tts
