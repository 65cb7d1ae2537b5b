// Rows to 8 bits (e4m3) with one scale per row and block of 128 columns:
//
//   scale = max(amax / 448, smallest normal float),   q = e4m3(value / scale)
//
// value is X, or silu(X[:, :n]) X[:, n:]; for dispatch, a token's row is quantised once and
// written to each of its pairs' rows. The largest magnitude of a block is a maximum over its lanes
// that keeps a NaN. The quotients are rounded as divisions are (a product with the reciprocal would
// round differently), at three instructions each.
//
// Bound by memory, but only just: some 25 (gated) instructions per element are 70 % of what the SMs
// can issue. Gated bf16 16384 x 2048: 30 us, 5.6 TB/s (with both operands unpacked as they arrive 37,
// with plain divisions, exponentials and 64-bit index arithmetic 74). Routed bf16 8192 x 4096 to 8
// experts each: 63 us, 5.5 TB/s (84 us); the scales' 4-byte writes land in rows far apart. Rows that
// do not start on 16 bytes take twice as long: 2047 columns gated 58 us.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cfloat>
#include "common.cuh"
#include "experts.h"
#include "values.cuh"

namespace appt {
namespace {

constexpr int kThreads = 256;

// How a block's columns lie in its lanes. kVec: 8 lanes of 16 neighbouring columns (32 bits: 16 lanes
// of 8), moved as 16-byte words. Else (rows that do not start on 16 bytes) 32 lanes of 4 neighbouring
// columns, read one by one, and stored as a word where rows of Q start on 4 bytes.
template <typename T, bool kVec>
struct Lay {
  static constexpr int kLanes = !kVec ? 32 : sizeof(T) == 4 ? 16 : 8;
  static constexpr int kPer = kScaleBlock / kLanes;
  static constexpr int kBlocksPerCta = kThreads / kLanes;
  // column of a lane's i-th value in the block
  static __device__ __forceinline__ int col(int lane, int i) { return lane * kPer + i; }
};

// A lane's values of a block of which the first n columns exist (kVec: all or none of a lane's),
// zeros for the others: fetched, and unpacked later, so that a gate and its factor are on their way
// together.
template <typename T, bool kVec>
struct Values {
  using L = Lay<T, kVec>;
  static constexpr int N = kVec ? 16 / sizeof(T) : 1;
  Pack<T, N> raw[L::kPer / N];
  __device__ __forceinline__ void fetch(const T* p, int lane, int n) {
#pragma unroll
    for (int i = 0; i < L::kPer / N; ++i) {
      raw[i] = Pack<T, N>{};
      if (L::col(lane, kVec ? 0 : i) < n) raw[i] = *(const Pack<T, N>*)(p + L::col(lane, i * N));
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[L::kPer]) const {
#pragma unroll
    for (int i = 0; i < L::kPer / N; ++i) {
      float f[N];
      raw[i].up(f);
#pragma unroll
      for (int k = 0; k < N; ++k) v[i * N + k] = f[k];
    }
  }
};

// x / s in fp32, rounded to nearest as a division is, for many x with one s: with y the rounded
// reciprocal and q = x y, one step q - (q s - x) y corrects the last place (Markstein's method; the
// remainder is exact in an fma). The remainder is taken with this sign because a zero's is then a
// zero whose product with -y has q's sign: -0 stays -0 (with x - q s it became +0). Holds while
// neither s, its reciprocal nor the remainder leaves the normal range; other scales (and those that
// are no numbers) divide.
struct Divisor {
  float s, y;
  __device__ __forceinline__ explicit Divisor(float scale) {
    s = scale;
    y = __frcp_rn(scale);
  }
  __device__ __forceinline__ bool holds() const { return s > 0x1p-60f && s < 0x1p60f; }
  __device__ __forceinline__ float of(float x) const {
    const float q = x * y;
    return __fmaf_rn(-__fmaf_rn(q, s, -x), y, q);
  }
};

// g / (1 + exp(-g)). 2^x and the reciprocal are the hardware's (2 steps and 1); the argument's
// rounding adds |g| 2^-24, which for g > 0 the 1 in the sum damps. Where exp(-g) passes 2^126 the
// reciprocal is 0, as 1 / infinity is a little further on.
__device__ __forceinline__ float silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}

// max(|a|, |b|, c), a NaN where one is
__device__ __forceinline__ float abs_max(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(c));
  return m;
}

struct Target {
  unsigned char* q;
  float* scale;
  long long cols;
  int ld, scale_ld, rows;
  bool words;   // rows of q start on 4 bytes
};

// A lane's 4 kWords values; words: rows of q start on 4 bytes (on 16 where kVec).
template <bool kVec, int kWords>
__device__ __forceinline__ void store_block(unsigned char* p, int lane, int n,
                                            const unsigned (&q)[kWords], bool words) {
  const int c = lane * 4 * kWords;
  if constexpr (kVec) {
    if (c >= n) return;
    if constexpr (kWords == 4) *(uint4*)(p + c) = make_uint4(q[0], q[1], q[2], q[3]);
    else *(uint2*)(p + c) = make_uint2(q[0], q[1]);
  } else if (words && c + 3 < n) {
    *(unsigned*)(p + c) = q[0];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < n) p[c + i] = (unsigned char)(q[0] >> (8 * i));
  }
}

__device__ __forceinline__ unsigned e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// kVec: every row of X (its gate's half too) and of Q starts on 16 bytes, and the columns are a
// multiple of 16. 2^groups_log2 groups of a block's lanes work on a row.
template <typename T, bool kGated, bool kRouted, bool kVec>
__global__ void __launch_bounds__(kThreads, 5)
    quantize_kernel(const T* __restrict__ x, long long ldx, long long rows,
                    const int* __restrict__ rows_ptr, const int* __restrict__ pair_row, int top_k,
                    int groups_log2, Target o) {
  using L = Lay<T, kVec>;
  constexpr int kPer = L::kPer;
  const int sub = threadIdx.x % L::kLanes, group = threadIdx.x / L::kLanes;
  // the block's lanes
  const unsigned mine = L::kLanes == 32
                            ? kFull
                            : ((1u << L::kLanes % 32) - 1) << (threadIdx.x & 31 & -L::kLanes);
  const int blocks = (int)((o.cols + kScaleBlock - 1) / kScaleBlock);
  const int step = 1 << groups_log2, per_cta = L::kBlocksPerCta >> groups_log2;
  if (!kRouted && rows_ptr) {
    const long long r = *rows_ptr;
    rows = r < rows ? (r > 0 ? r : 0) : rows;
  }
  for (long long row = (long long)blockIdx.x * per_cta + (group >> groups_log2); row < rows;
       row += (long long)gridDim.x * per_cta) {
    for (int block = group & (step - 1); block < blocks; block += step) {
      const long long col = (long long)block * kScaleBlock;
      const int n = o.cols - col < kScaleBlock ? (int)(o.cols - col) : kScaleBlock;
      const T* p = x + row * ldx + col;
      Values<T, kVec> in, factor;
      in.fetch(p, sub, n);
      if (kGated) factor.fetch(p + o.cols, sub, n);
      float v[kPer];
      in.unpack(v);
      if (kGated) {
        float up[kPer];
        factor.unpack(up);
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = silu(v[k]) * up[k];
      }
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < kPer; k += 2) top = abs_max(v[k], v[k + 1], top);
#pragma unroll
      for (int s = L::kLanes / 2; s > 0; s >>= 1)
        top = abs_max(__shfl_xor_sync(mine, top, s), 0.f, top);
      float scale = __fdiv_rn(top, 448.f);
      if (scale < FLT_MIN) scale = FLT_MIN;   // false for NaN
      const Divisor div(scale);
      unsigned q[kPer / 4];
      if (div.holds()) {
#pragma unroll
        for (int k = 0; k < kPer / 4; ++k)
          q[k] = e4m3x2(div.of(v[4 * k]), div.of(v[4 * k + 1])) |
                 e4m3x2(div.of(v[4 * k + 2]), div.of(v[4 * k + 3])) << 16;
      } else {
#pragma unroll
        for (int k = 0; k < kPer / 4; ++k)
          q[k] = e4m3x2(__fdiv_rn(v[4 * k], scale), __fdiv_rn(v[4 * k + 1], scale)) |
                 e4m3x2(__fdiv_rn(v[4 * k + 2], scale), __fdiv_rn(v[4 * k + 3], scale)) << 16;
      }
      float* ps = o.scale + (long long)block * o.scale_ld;
      if (kRouted) {
        const int* pr = pair_row + row * top_k;
        unsigned char* pq = o.q + col;
        for (int j0 = 0; j0 < top_k; j0 += 4) {
          int r[4];   // on their way together
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = j0 + j < top_k ? pr[j0 + j] : -1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if ((unsigned)r[j] >= (unsigned)o.rows) continue;
            store_block<kVec>(pq + (long long)r[j] * o.ld, sub, n, q, o.words);
            if (sub == 0) ps[r[j]] = scale;
          }
        }
      } else {
        store_block<kVec>(o.q + row * o.ld + col, sub, n, q, o.words);
        if (sub == 0) ps[row] = scale;
      }
    }
  }
}

template <typename T, bool kVec>
void quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
              const Target& o, cudaStream_t s) {
  const long long blocks = (o.cols + kScaleBlock - 1) / kScaleBlock;
  int groups = 0;   // no more than a row has blocks
  constexpr int kBlocksPerCta = Lay<T, kVec>::kBlocksPerCta;
  while (2 << groups <= kBlocksPerCta && 2 << groups <= blocks) ++groups;
  const int per_cta = kBlocksPerCta >> groups;
  const long long ctas = (x.rows + per_cta - 1) / per_cta;
  const dim3 grid((unsigned)(ctas < (1 << 20) ? ctas : 1 << 20));
  const T* p = (const T*)x.data;
  if (routes)
    launch(nullptr, quantize_kernel<T, false, true, kVec>, grid, kThreads, 0, s, 1, p, x.ld, x.rows,
           nullptr, routes->pair_row, routes->top_k, groups, o);
  else if (gated)
    launch(nullptr, quantize_kernel<T, true, false, kVec>, grid, kThreads, 0, s, 1, p, x.ld, x.rows,
           rows_ptr, nullptr, 1, groups, o);
  else
    launch(nullptr, quantize_kernel<T, false, false, kVec>, grid, kThreads, 0, s, 1, p, x.ld,
           x.rows, rows_ptr, nullptr, 1, groups, o);
}

template <typename T>
void quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
              const Target& o, cudaStream_t s) {
  const bool vec = (uintptr_t)x.data % 16 == 0 && x.ld * sizeof(T) % 16 == 0 &&
                   (uintptr_t)o.q % 16 == 0 && o.ld % 16 == 0 && o.cols % 16 == 0;
  if (vec) quantize<T, true>(x, gated, rows_ptr, routes, o, s);
  else quantize<T, false>(x, gated, rows_ptr, routes, o, s);
}

}  // namespace

int launch_quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
                    const ScaledView& q, cudaStream_t s) {
  if (x.rows == 0 || q.q.cols == 0 || q.q.rows == 0) return 0;
  const Target o{(unsigned char*)q.q.data, q.scale, q.q.cols, (int)q.q.ld, (int)q.scale_ld,
                 (int)q.q.rows, (uintptr_t)q.q.data % 4 == 0 && q.q.ld % 4 == 0};
  switch (x.type) {
    case kF32: quantize<float>(x, gated, rows_ptr, routes, o, s); break;
    case kF16: quantize<__half>(x, gated, rows_ptr, routes, o, s); break;
    default: quantize<__nv_bfloat16>(x, gated, rows_ptr, routes, o, s); break;
  }
  return 1;
}

}  // namespace appt
