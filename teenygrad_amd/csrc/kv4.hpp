// Lanes of a row of 16 that hold a token each: kv4_cache.hip and kv4_attn.hip.
#pragma once

#include "mfma.hpp"

#include <type_traits>
#include <utility>

namespace teeny {

int kv_page_shift(int64_t page_size);

// v of lane I of the row of 16 lanes (row_newbcast)
template <int I>
__device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xf, 0xf, true));
}

// f(std::integral_constant<int, 0>) .. f(std::integral_constant<int, 15>)
template <typename F, int... I>
__device__ __forceinline__ void each16(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <typename F>
__device__ __forceinline__ void each16(F f) {
  each16(f, std::make_integer_sequence<int, 16>{});
}

}  // namespace teeny
