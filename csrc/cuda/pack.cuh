// Vector accesses with conversion to and from fp32 (decoder-block kernels).
#pragma once
#include <type_traits>

#include "common.cuh"

namespace nexar {

// W elements of T (bf16, fp16 or fp32; W even), read and written in up to
// 16-byte accesses and kept as words until they are needed. Conversions to 16
// bits go two at a time: one at a time they run on the SM's narrowest pipe
// (dropout of 64 Mi bf16 elements: 60 us, two at a time 49).
template <typename T, int W> struct alignas(W * sizeof(T) < 16 ? W * sizeof(T) : 16) Pack {
  static constexpr int kWords = W * sizeof(T) / 4;
  uint32_t w[kWords];
  NEXAR_D void load(const T* p) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      *this = *reinterpret_cast<const Pack*>(p);
    }
  }
  NEXAR_D void store(T* p) const { *reinterpret_cast<Pack*>(p) = *this; }
  NEXAR_D float2 get(int pair) const {  // elements 2 pair, 2 pair + 1
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * pair]), __uint_as_float(w[2 * pair + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w[pair]));
    else return make_float2(__uint_as_float(w[pair] << 16), __uint_as_float(w[pair] & 0xffff0000u));
  }
  NEXAR_D void set(int pair, float lo, float hi) {
    if constexpr (sizeof(T) == 4) {
      w[2 * pair] = __float_as_uint(lo), w[2 * pair + 1] = __float_as_uint(hi);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 v = __floats2half2_rn(lo, hi);
      w[pair] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      w[pair] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
};

}  // namespace nexar
