// Element types of the routed products' dense operands: their accumulator type, conversion, and
// 16-byte vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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

// N consecutive elements, moved as one access.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

}  // namespace appt
