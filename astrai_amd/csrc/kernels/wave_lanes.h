// Reductions over groups of 16, 32 or 64 lanes by cross-lane moves of the vector unit
// (DPP and permlane swaps): a step takes an instruction, where a shuffle is a trip
// through LDS of a hundred cycles and more.
#pragma once

#include "moe_common.h"

namespace astrai_moe {
namespace {

template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// v of the lane that STEP says: 0, 1: 1 and 2 lanes apart; 2, 3: the halves of 8 and of
// 16 mirrored; 4, 5: the other 16-lane row, the other 32-lane half (once v is alike
// within these).
template <int STEP>
__device__ __forceinline__ unsigned other(unsigned v) {
  if constexpr (STEP < 4) {
    return dpp<STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140>(v);
  } else {
    const auto r = [&] {
      if constexpr (STEP == 4)
        return __builtin_amdgcn_permlane16_swap(v, v, false, false);
      else
        return __builtin_amdgcn_permlane32_swap(v, v, false, false);
    }();
    return r[0] ^ r[1] ^ v;  // (one of them is the lane's own)
  }
}
template <int STEP>
__device__ __forceinline__ int other(int v) {
  return (int)other<STEP>((unsigned)v);
}
template <int STEP>
__device__ __forceinline__ float other(float v) {
  return __builtin_bit_cast(float, other<STEP>(__builtin_bit_cast(unsigned, v)));
}
template <int STEP>
__device__ __forceinline__ uint64_t other(uint64_t v) {
  return (uint64_t)other<STEP>((unsigned)(v >> 32)) << 32 | other<STEP>((unsigned)v);
}
template <int STEP>
__device__ __forceinline__ double other(double v) {
  return __builtin_bit_cast(double, other<STEP>(__builtin_bit_cast(uint64_t, v)));
}

// op over groups of L lanes, in every one of them. Needs the whole wave.
template <int L, typename F, typename Op>
__device__ __forceinline__ F reduce(F v, Op op) {
  v = op(v, other<0>(v));
  v = op(v, other<1>(v));
  v = op(v, other<2>(v));
  v = op(v, other<3>(v));
  if constexpr (L >= 32) v = op(v, other<4>(v));
  if constexpr (L >= 64) v = op(v, other<5>(v));
  return v;
}
template <int L, typename F>
__device__ __forceinline__ F lanes_max(F v) {
  return reduce<L>(v, [](F a, F b) { return a > b ? a : b; });
}
template <int L, typename F>
__device__ __forceinline__ F lanes_sum(F v) {
  return reduce<L>(v, [](F a, F b) { return a + b; });
}

}  // namespace
}  // namespace astrai_moe
