// Element types of the routed products' dense operands: their accumulator type, conversion, and
// 16-byte vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <type_traits>

namespace appt {

template <typename T> struct Value {             // fp32
  using Acc = float;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Value<double> {
  using Acc = double;
  static __device__ __forceinline__ double up(double x) { return x; }
  static __device__ __forceinline__ double down(double x) { return x; }
};
template <> struct Value<__half> {
  using Acc = float;
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Value<__nv_bfloat16> {
  using Acc = float;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

// N consecutive elements moved as one access: one element, or 4, 8 or 16 bytes kept as words
// (arrays of 16-bit elements would take a register each).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  using A = typename Value<T>::Acc;
  static constexpr int kWords = sizeof(T) * N / 4;
  unsigned word[kWords];
  __device__ __forceinline__ void up(A (&v)[N]) const {
    if constexpr (sizeof(T) == 8) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = __hiloint2double((int)word[2 * i + 1], (int)word[2 * i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 4) {
          v[i] = __uint_as_float(word[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2_raw r{(unsigned short)word[i], (unsigned short)(word[i] >> 16)};
          const float2 f = __half22float2(__half2(r));
          v[2 * i] = f.x, v[2 * i + 1] = f.y;
        } else {   // bf16 is the upper half of fp32
          v[2 * i] = __uint_as_float(word[i] << 16);
          v[2 * i + 1] = __uint_as_float(word[i] & 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ void down(const A (&v)[N]) {
    if constexpr (sizeof(T) == 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        word[2 * i] = (unsigned)__double2loint(v[i]);
        word[2 * i + 1] = (unsigned)__double2hiint(v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 4) {
          word[i] = __float_as_uint(v[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2_raw r(__floats2half2_rn(v[2 * i], v[2 * i + 1]));
          word[i] = r.x | (unsigned)r.y << 16;
        } else {
          const __nv_bfloat162_raw r(__floats2bfloat162_rn(v[2 * i], v[2 * i + 1]));
          word[i] = r.x | (unsigned)r.y << 16;
        }
      }
    }
  }
};
template <typename T>
struct Pack<T, 1> {
  using A = typename Value<T>::Acc;
  T w;
  __device__ __forceinline__ void up(A (&v)[1]) const { v[0] = Value<T>::up(w); }
  __device__ __forceinline__ void down(const A (&v)[1]) { w = Value<T>::down(v[0]); }
};

}  // namespace appt
