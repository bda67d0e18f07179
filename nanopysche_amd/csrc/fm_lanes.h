// Sums and other folds over groups of neighbouring lanes, without LDS: moves within rows of 16 lanes, then the
// swaps of rows and halves.
#pragma once

#include <type_traits>

#include "fm_tile.h"

namespace fm {

// lanes of a group of N (a power of two) folded by f, and their sum: the same in every lane
template <int N, typename F>
__device__ __forceinline__ float group_fold(float v, F f) {
  auto dpp = [](float x, auto ctrl) { return __builtin_bit_cast(float, dpp_move<decltype(ctrl)::value>(__builtin_bit_cast(int, x))); };
  if constexpr (N > 1) v = f(v, dpp(v, std::integral_constant<int, kDppQuadSwap1>{}));
  if constexpr (N > 2) v = f(v, dpp(v, std::integral_constant<int, kDppQuadSwap2>{}));
  if constexpr (N > 4) v = f(v, dpp(v, std::integral_constant<int, kDppRowHalfMirror>{}));
  if constexpr (N > 8) v = f(v, dpp(v, std::integral_constant<int, kDppRowRor8>{}));
  if constexpr (N > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    v = f(u2f(a[0]), u2f(a[1]));
  }
  if constexpr (N > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = f(u2f(a[0]), u2f(a[1]));
  }
  return v;
}
template <int N>
__device__ __forceinline__ float group_sum(float v) {
  return group_fold<N>(v, [](float a, float b) { return a + b; });
}

}  // namespace fm
