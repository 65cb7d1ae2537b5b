// Products of rows in 8 bits with each group's matrix in 8 bits, scales by blocks of 128:
//
//   Y[r, n] = sum_b sa[b, r] sw[g, n / 128, b] sum_{k in block b} a[r, k] w[g, n, k]
//
// for the rows r of group g. Sums in fp32.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include "common.cuh"
#include "experts.h"
#include "values.cuh"

namespace appt {
namespace {

constexpr int kTile = 32;    // rows and columns of Y per CTA

__device__ __forceinline__ float e4m3(unsigned char x) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
}

template <typename T>
__global__ void __launch_bounds__(256)
    product_kernel(const unsigned char* a, long long lda, const float* sa, long long lds,
                   int rows, const unsigned char* w, long long ldw, long long group_stride,
                   const float* sw, int groups, int n_rows, int cols, const int* group_ptr, T* y,
                   long long ldy) {
  __shared__ float ta[kTile][kTile + 1], tw[kTile][kTile + 1];
  const int nb = (cols + kScaleBlock - 1) / kScaleBlock;
  const int nn = (n_rows + kScaleBlock - 1) / kScaleBlock;
  const int n0 = blockIdx.x * kTile, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int g = blockIdx.y; g < groups; g += gridDim.y) {
    const int r_lo = group_ptr ? max(0, min(group_ptr[g], rows)) : 0;
    const int r_hi = group_ptr ? max(r_lo, min(group_ptr[g + 1], rows)) : rows;
    for (int r0 = r_lo + blockIdx.z * kTile; r0 < r_hi; r0 += gridDim.z * kTile) {
      float sum[4] = {0, 0, 0, 0};
      for (int k0 = 0; k0 < cols; k0 += kTile) {
        const int k = k0 + tx, b = k0 / kScaleBlock;
        for (int i = ty; i < kTile; i += 8) {
          const int r = r0 + i, n = n0 + i;
          ta[i][tx] = r < r_hi && k < cols ? e4m3(a[r * lda + k]) * sa[b * lds + r] : 0.f;
          tw[i][tx] = n < n_rows && k < cols
                          ? e4m3(w[g * group_stride + n * ldw + k]) *
                                sw[((long long)g * nn + n / kScaleBlock) * nb + b]
                          : 0.f;
        }
        __syncthreads();
        for (int k1 = 0; k1 < kTile; ++k1)
          for (int i = 0; i < 4; ++i) sum[i] += ta[ty + 8 * i][k1] * tw[tx][k1];
        __syncthreads();
      }
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + ty + 8 * i, n = n0 + tx;
        if (r < r_hi && n < n_rows) y[r * ldy + n] = Value<T>::down(sum[i]);
      }
    }
  }
}

template <typename T>
void product(const ScaledView& a, const BlocksView& w, const int* group_ptr, const DenseView& y,
             cudaStream_t s) {
  const dim3 grid((unsigned)((w.rows + kTile - 1) / kTile), (unsigned)w.groups,
                  (unsigned)min((y.rows + kTile - 1) / kTile, 64ll));
  launch(nullptr, product_kernel<T>, grid, 256, 0, s, (const unsigned char*)a.q.data, a.q.ld,
         a.scale, a.scale_ld, (int)a.q.rows, (const unsigned char*)w.data, w.ld, w.group_stride,
         w.scale, (int)w.groups, (int)w.rows, (int)w.cols, group_ptr, (T*)y.data, y.ld);
}

}  // namespace

int launch_scaled_product(const ScaledView& a, const BlocksView& w, const int* group_ptr,
                          const DenseView& y, int sms, cudaStream_t s) {
  (void)sms;
  switch (y.type) {
    case kF32: product<float>(a, w, group_ptr, y, s); break;
    case kF16: product<__half>(a, w, group_ptr, y, s); break;
    default: product<__nv_bfloat16>(a, w, group_ptr, y, s); break;
  }
  return 1;
}

}  // namespace appt
