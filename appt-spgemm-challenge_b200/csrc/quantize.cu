// Rows to 8 bits (e4m3) with one scale per row and block of 128 columns:
//
//   scale = max(amax / 448, smallest normal float),   q = e4m3(value / scale)
//
// value is X, or silu(X[:, :n]) X[:, n:]; for dispatch, a token's row is quantised once and
// written to each of its pairs' rows. 16 lanes hold a block, 8 neighbouring columns each; the
// largest magnitude is a maximum of the bit patterns without sign, in which a NaN is above
// infinity, so neither is lost. Bound by memory: the quotients are true divisions (a product with
// the reciprocal rounds differently), some 10 instructions per element and still below the copy.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cfloat>
#include "common.cuh"
#include "experts.h"
#include "values.cuh"

namespace appt {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerCta = kThreads / 16;   // scale blocks that a CTA holds at a time

template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float v[8]) {
  if (vec && n >= 8) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const Pack<T, N> x = *(const Pack<T, N>*)(p + i);
#pragma unroll
      for (int k = 0; k < N; ++k) v[i + k] = Value<T>::up(x.v[k]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Value<T>::up(p[i]) : 0.f;
  }
}

struct Target {
  unsigned char* q;
  long long ld;
  float* scale;
  long long scale_ld;
  long long rows, cols;
  bool vec;             // rows of q start on 8 bytes
};

__device__ __forceinline__ void store8(const Target& o, long long row, long long col, int n,
                                       uint2 q) {
  unsigned char* p = o.q + row * o.ld + col;
  if (o.vec && n >= 8) {
    *(uint2*)p = q;
  } else {
    const unsigned long long both = (unsigned long long)q.y << 32 | q.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (unsigned char)(both >> (8 * i));
  }
}

template <typename T, bool kGated, bool kRouted>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(const T* __restrict__ x, long long ldx, bool xvec, long long rows,
                    const int* __restrict__ rows_ptr, const int* __restrict__ pair_row, int top_k,
                    Target o) {
  const int sub = threadIdx.x & 15;
  const long long blocks = (o.cols + kScaleBlock - 1) / kScaleBlock;
  if (!kRouted && rows_ptr) {
    const long long r = *rows_ptr;
    rows = r < rows ? (r > 0 ? r : 0) : rows;
  }
  const long long items = rows * blocks;   // (row, block), blocks of a row next to each other
  const long long step = (long long)gridDim.x * kBlocksPerCta;
  // whole warps run the loop: the two halves' items differ by one
  for (long long i0 = (long long)blockIdx.x * kBlocksPerCta + (threadIdx.x >> 5) * 2; i0 < items;
       i0 += step) {
    const long long i = i0 + ((threadIdx.x >> 4) & 1);
    const bool on = i < items;
    const long long row = on ? i / blocks : 0, block = on ? i % blocks : 0;
    const long long col = block * kScaleBlock + sub * 8;
    const int n = on ? (int)(o.cols - col < 8 ? (o.cols > col ? o.cols - col : 0) : 8) : 0;
    float v[8];
    const T* p = x + row * ldx + col;
    load8(p, n, xvec, v);
    if (kGated) {
      float u[8];
      load8(p + o.cols, n, xvec && o.cols % (16 / (int)sizeof(T)) == 0, u);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = v[k] / (1.f + expf(-v[k])) * u[k];
    }
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(kFull, top, s));
    float scale = __fdiv_rn(__uint_as_float(top), 448.f);
    if (scale < FLT_MIN) scale = FLT_MIN;   // false for NaN
    unsigned q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      q[k] = __nv_cvt_float2_to_fp8x2(
          make_float2(__fdiv_rn(v[2 * k], scale), __fdiv_rn(v[2 * k + 1], scale)), __NV_SATFINITE,
          __NV_E4M3);
    const uint2 out = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    if (kRouted) {
      if (!on) continue;
      for (int j = 0; j < top_k; ++j) {
        const int r = pair_row[row * top_k + j];
        if (r < 0 || r >= o.rows) continue;
        store8(o, r, col, n, out);
        if (sub == 0) o.scale[block * o.scale_ld + r] = scale;
      }
    } else if (on) {
      store8(o, row, col, n, out);
      if (sub == 0) o.scale[block * o.scale_ld + row] = scale;
    }
  }
}

template <typename T>
void quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
              const Target& o, cudaStream_t s) {
  const bool xvec = (uintptr_t)x.data % 16 == 0 && x.ld * sizeof(T) % 16 == 0;
  const long long items = x.rows * ((o.cols + kScaleBlock - 1) / kScaleBlock);
  const long long ctas = (items + kBlocksPerCta - 1) / kBlocksPerCta;
  const dim3 grid((unsigned)(ctas < (1 << 20) ? ctas : 1 << 20));
  const T* p = (const T*)x.data;
  if (routes)
    launch(nullptr, quantize_kernel<T, false, true>, grid, kThreads, 0, s, 1, p, x.ld, xvec, x.rows,
           nullptr, routes->pair_row, routes->top_k, o);
  else if (gated)
    launch(nullptr, quantize_kernel<T, true, false>, grid, kThreads, 0, s, 1, p, x.ld, xvec, x.rows,
           rows_ptr, nullptr, 1, o);
  else
    launch(nullptr, quantize_kernel<T, false, false>, grid, kThreads, 0, s, 1, p, x.ld, xvec, x.rows,
           rows_ptr, nullptr, 1, o);
}

}  // namespace

int launch_quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
                    const ScaledView& q, cudaStream_t s) {
  if (x.rows == 0 || q.q.cols == 0 || q.q.rows == 0) return 0;
  const Target o{(unsigned char*)q.q.data, q.q.ld, q.scale, q.scale_ld, q.q.rows, q.q.cols,
                 (uintptr_t)q.q.data % 8 == 0 && q.q.ld % 8 == 0};
  switch (x.type) {
    case kF32: quantize<float>(x, gated, rows_ptr, routes, o, s); break;
    case kF16: quantize<__half>(x, gated, rows_ptr, routes, o, s); break;
    default: quantize<__nv_bfloat16>(x, gated, rows_ptr, routes, o, s); break;
  }
  return 1;
}

}  // namespace appt
