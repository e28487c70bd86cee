// Reductions over neighbouring lanes, shared by the operators' kernels.
#pragma once
#include <hip/hip_runtime.h>

namespace tts {

template <int CTRL, class T>
__device__ __forceinline__ T dpp_moved(T v) {
  static_assert(sizeof(T) == 4, "");
  const int d = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, d, CTRL, 0xf, 0xf, true));  // (0 where there is no such lane)
}

// f over groups of G neighbouring lanes, in all of them: up to 16 lanes by DPP moves, which read lanes of the group alone
template <int G, class T, class F>
__device__ __forceinline__ T over_lanes(T v, F f) {
  if constexpr (G > 1) v = f(v, dpp_moved<0xb1>(v));   // quad_perm [1, 0, 3, 2]
  if constexpr (G > 2) v = f(v, dpp_moved<0x4e>(v));   // quad_perm [2, 3, 0, 1]
  if constexpr (G > 4) v = f(v, dpp_moved<0x141>(v));  // row_half_mirror: the other four
  if constexpr (G > 8) v = f(v, dpp_moved<0x128>(v));  // row_ror 8: the other eight
  if constexpr (G > 16) v = f(v, __shfl_xor(v, 16));
  if constexpr (G > 32) v = f(v, __shfl_xor(v, 32));
  return v;
}

}  // namespace tts
