// Tables and rows of values in fp32, bf16 or fp16: computed with in fp32, rounded once when written.
#pragma once

#include "slg_common.h"

namespace slg {

enum { kTabF32 = 0, kTabBf16 = 1, kTabF16 = 2 };

template <int DT> struct TabType;
template <> struct TabType<kTabF32> { using t = float; };
template <> struct TabType<kTabBf16> { using t = uint16_t; };
template <> struct TabType<kTabF16> { using t = _Float16; };

template <int DT>
__device__ inline float tab_get(typename TabType<DT>::t v) {
  if constexpr (DT == kTabBf16) return __uint_as_float((uint32_t)v << 16);
  else return (float)v;
}

// Round to nearest even; a NaN stays one.
template <int DT>
__device__ inline typename TabType<DT>::t tab_put(float v) {
  if constexpr (DT == kTabBf16) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
  } else {
    return (typename TabType<DT>::t)v;
  }
}

}  // namespace slg
