// mla_elem.h -- element types of the kernels around the decode: values, and 16 bytes of them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mla_srv {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Bf16 {
  static constexpr int kBytes = 2;
  typedef uint16_t bits;
  __device__ static float value(bits b) { return __uint_as_float((uint32_t)b << 16); }
  __device__ static bits of(float v) { return __builtin_bit_cast(bits, (__bf16)v); }
};
struct F16 {
  static constexpr int kBytes = 2;
  typedef uint16_t bits;
  __device__ static float value(bits b) { return (float)__builtin_bit_cast(_Float16, b); }
  __device__ static bits of(float v) { return __builtin_bit_cast(bits, (_Float16)v); }
};
struct F32 {
  static constexpr int kBytes = 4;
  typedef uint32_t bits;
  __device__ static float value(bits b) { return __uint_as_float(b); }
  __device__ static bits of(float v) { return __float_as_uint(v); }
};

// 16 bytes to floats and back (8 values, or 4 of fp32)
template <class E>
__device__ __forceinline__ void unpack(const i32x4 v, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (uint32_t)v[j];
    if constexpr (E::kBytes == 4) {
      x[j] = __uint_as_float(w);
    } else if constexpr (__is_same(E, Bf16)) {
      x[2 * j] = __uint_as_float(w << 16);
      x[2 * j + 1] = __uint_as_float(w & 0xFFFF0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * j] = (float)h[0];
      x[2 * j + 1] = (float)h[1];
    }
  }
}
template <class E>
__device__ __forceinline__ i32x4 pack(const float* x) {
  i32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (E::kBytes == 4)
      v[j] = (int)__float_as_uint(x[j]);
    else if constexpr (__is_same(E, Bf16))
      v[j] = __builtin_bit_cast(int, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), bf16x2));
    else
      v[j] = __builtin_bit_cast(int, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), f16x2));
  }
  return v;
}

}  // namespace mla_srv
