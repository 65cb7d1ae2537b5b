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
// can issue. Gated bf16 16384 x 2048: 31 us, 5.5 TB/s (with both operands unpacked as they arrive 37,
// with plain divisions, exponentials and 64-bit index arithmetic 74). Routed bf16 8192 x 4096 to 8
// experts each: 63 us, 5.5 TB/s (84 us); the scales' 4-byte writes land in rows far apart. Rows that
// do not start on 16 bytes take twice as long: 2047 columns gated 59 us.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cfloat>
#include "common.cuh"
#include "experts.h"
#include "tcgen05.cuh"
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

// v = silu(v) up, in pairs of neighbours: silu(g) = g / (1 + exp(-g)), below 10 half steps of fp32
// with the product. 2^x and the reciprocal are the hardware's (2 steps and 1). The argument
// -g log2(e) rounded would alone be off by |g| half steps (5e-6 at -80), so x and m have exp(-g) =
// 2^x exp(m), m small. For 16-bit gates x is an exact product with the leading bits of log2(e) and m
// the other bits' part; for bf16 1 + m is exp(m) but for m^2 / 2 (half a step more at -50, 1.3 at
// -80), for fp16 the square is taken too. Else m is what rounding took from x, and exp(m) = 1 + m.
// No branch: gates below -87.3, whose silu is smaller than 2^-119, get a reciprocal of 0 and with it
// a 0; and an infinite gate's 0 times m is a NaN, which a maximum with 1, never above 1 + exp(-g),
// takes away (a gate that is a NaN is a factor still). A way of its own for far gates, to where silu
// leaves fp32 near -104, took 33 to 39 us instead of 31 even where there was none, for it cuts the
// block's instructions in two.
template <typename T>
__device__ __forceinline__ void gate(float& v0, float& v1, float up0, float up1) {
  using namespace sm100;
  const uint64_t g = two(v0, v1);
  uint64_t m;
  float e0, e1;
  if constexpr (sizeof(T) == 2) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kLog2e = kHalf ? 0x1.715p+0f : 0x1.7154p+0f;        // 13 and 15 bits
    // the other bits, times -ln(2)
    constexpr float kRestLn2 = kHalf ? -0x1.8be626p-15f : -0x1.480fb6p-18f;
    untwo(mul_two(g, two(-kLog2e, -kLog2e)), e0, e1);
    m = mul_two(g, two(kRestLn2, kRestLn2));
    if (kHalf) m = mul_two(m, fma_two(m, two(0.5f, 0.5f), two(1.f, 1.f)));
  } else {
    constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0cp-26f;   // their sum: log2(e)
    constexpr float kLn2 = 0x1.62e43p-1f;
    untwo(mul_two(g, two(-kLog2e, -kLog2e)), e0, e1);
    e0 = fminf(e0, 127.f), e1 = fminf(e1, 127.f);   // no infinity times a negative m
    m = fma_two(g, two(kLog2e, kLog2e), two(e0, e1));   // exact
    m = fma_two(g, two(kRest, kRest), m);
    m = mul_two(m, two(-kLn2, -kLn2));
  }
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
  const uint64_t e = two(e0, e1);
  untwo(add_two(fma_two(e, m, e), two(1.f, 1.f)), e0, e1);
  e0 = fmaxf(e0, 1.f), e1 = fmaxf(e1, 1.f);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
  untwo(mul_two(mul_two(g, two(e0, e1)), two(up0, up1)), v0, v1);
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
        for (int k = 0; k < kPer; k += 2) gate<T>(v[k], v[k + 1], up[k], up[k + 1]);
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
