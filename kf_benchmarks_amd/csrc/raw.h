// V neighbouring values as loaded, kept packed until they are used: an array of
// 16-bit elements would be given a register each.
#pragma once
#include "common.h"

namespace kfb {

template <typename T, int V> struct Raw {
  static constexpr int ND = (V * (int)sizeof(T) + 3) / 4;
  uint32_t d[ND];

  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (V * sizeof(T) == 16) {
      typedef __attribute__((ext_vector_type(4))) uint32_t u4;
      const u4 q = *(const u4*)p;
      d[0] = q.x; d[1] = q.y; d[2] = q.z; d[3] = q.w;
    } else if constexpr (V * sizeof(T) == 8) {
      typedef __attribute__((ext_vector_type(2))) uint32_t u2;
      const u2 q = *(const u2*)p;
      d[0] = q.x; d[1] = q.y;
    } else if constexpr (V * sizeof(T) == 4) {
      d[0] = *(const uint32_t*)p;
    } else {
      static_assert(V == 1 && sizeof(T) == 2, "16, 8, 4 or 2 bytes");
      d[0] = *(const uint16_t*)p;
    }
  }

  // zero unless ``on``
  __device__ __forceinline__ void keep(bool on) {
#pragma unroll
    for (int i = 0; i < ND; ++i) d[i] = on ? d[i] : 0;
  }

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < ND; ++i) d[i] = 0;
  }

  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, d[i]);
    else if constexpr (__is_same(T, bf16))
      return __builtin_bit_cast(float, i & 1 ? d[i / 2] & 0xffff0000u : d[i / 2] << 16);
    else return (float)__builtin_bit_cast(f16, (uint16_t)(d[i / 2] >> (16 * (i & 1))));
  }
};

}  // namespace kfb
