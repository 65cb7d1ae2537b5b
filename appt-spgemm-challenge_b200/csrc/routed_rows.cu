// Dense rows to the experts' order and back: the products of the routing matrix R (tokens x
// sorted rows, weights as entries) with dense matrices.
//
//   dispatch      Y = R^T X          Y[row(p)] = w[p] X[p / k]
//   combine       Y = R H            Y[t] = sum_j w[t,j] H[row(t,j)]
//   combine_grad  dH = R^T dY, and the sampled product dw[p] = <dY[p / k], H[row(p)]>
//
// All are bound by memory: a few operations per element. Each goes by tokens, so that a token's
// row is read (or written) once for its k pairs, and each thread moves 16-byte pieces (8, 4 or one
// element's bytes where rows do not start on 16). Measured with 4,096 columns of bf16: dispatch of
// 8,192 tokens to 8 experts 96 us, 6.3 TB/s; gradient of combine with 4 experts 94 us, 6.1 TB/s
// (106 us at three CTAs per SM instead of four); combine of 32 tokens of 8 (fp16) 2.6 us. 1,111
// columns of fp32, 1,000 tokens to 3 experts, move element by element: 5.4 us, 3.1 TB/s.
#include <cuda_runtime.h>
#include <algorithm>
#include "common.cuh"
#include "experts.h"
#include "values.cuh"

namespace appt {
namespace {

constexpr int kThreads = 256;

// Pieces that a thread has in flight. A piece is 16 bytes, or 8 or 4 or a single element where rows
// do not start and end on 16 bytes: more of those.
__host__ __device__ constexpr int dispatch_pieces(int bytes) { return bytes == 16 ? 4 : 8; }
__host__ __device__ constexpr int combine_pieces(int bytes) { return bytes == 16 ? 1 : 4; }

// What the three kernels share: `lanes` (a multiple of 32) threads per token.
struct Shape {
  const int* pair_row;
  int tokens, top_k;
  int pieces;           // pieces of N elements per row
  int lanes;
};

struct Place {
  int token;            // -1: none
  int at;               // thread's place among the token's
};

__device__ __forceinline__ Place place(const Shape& s) {
  const int per = kThreads / s.lanes;
  const long long t = (long long)blockIdx.x * per + threadIdx.x / s.lanes;
  return Place{t < s.tokens ? (int)t : -1, (int)threadIdx.x % s.lanes};
}

// Rows (-1: dropped or out of range) of up to 32 pairs of a token, one per lane.
__device__ __forceinline__ int lane_row(const Shape& s, int token, int j0, int rows) {
  const int j = j0 + (threadIdx.x & 31);
  const int r = j < s.top_k ? s.pair_row[(long long)token * s.top_k + j] : -1;
  return r >= 0 && r < rows ? r : -1;
}

template <typename A>
__device__ __forceinline__ A lane_weight(const Shape& s, const A* w, int token, int j0, int row) {
  return w && row >= 0 ? w[(long long)token * s.top_k + j0 + (threadIdx.x & 31)] : A(1);
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
    dispatch_kernel(Shape s, const T* __restrict__ x, int ldx,
                    const typename Value<T>::Acc* __restrict__ w, T* __restrict__ y, int ldy,
                    int rows) {
  using A = typename Value<T>::Acc;
  using P = Pack<T, N>;
  constexpr int U = dispatch_pieces(N * sizeof(T));
  const Place me = place(s);
  if (me.token < 0) return;   // whole warps
  const P* px = (const P*)(x + (long long)me.token * ldx);
  // (64-bit: past the last piece of a long row, 32 bits could wrap)
  for (long long base = (long long)blockIdx.y * s.lanes * U; base < s.pieces;
       base += (long long)gridDim.y * s.lanes * U) {
    P v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long c = base + me.at + (long long)u * s.lanes;
      if (c < s.pieces) v[u] = px[c];
    }
    for (int j0 = 0; j0 < s.top_k; j0 += 32) {
      const int mine = lane_row(s, me.token, j0, rows);
      const A wmine = lane_weight(s, w, me.token, j0, mine);
      for (int j = 0; j < 32 && j0 + j < s.top_k; ++j) {
        const int row = __shfl_sync(kFull, mine, j);
        const A wj = __shfl_sync(kFull, wmine, j);
        if (row < 0) continue;
        P* py = (P*)(y + (long long)row * ldy);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const long long c = base + me.at + (long long)u * s.lanes;
          if (c >= s.pieces) continue;
          P o = v[u];
          if (w) {
            A f[N];
            v[u].up(f);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] *= wj;
            o.down(f);
          }
          py[c] = o;
        }
      }
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
    combine_kernel(Shape s, const T* __restrict__ h, int ldh, int rows,
                   const typename Value<T>::Acc* __restrict__ w, T* __restrict__ y, int ldy) {
  using A = typename Value<T>::Acc;
  using P = Pack<T, N>;
  constexpr int J = 4;   // rows in flight
  constexpr int U = combine_pieces(N * sizeof(T));
  const Place me = place(s);
  if (me.token < 0) return;
  P* py = (P*)(y + (long long)me.token * ldy);
  for (long long base = (long long)blockIdx.y * s.lanes * U; base < s.pieces;
       base += (long long)gridDim.y * s.lanes * U) {
    const long long c0 = base + me.at;
    A sum[U][N];
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) sum[k][i] = A(0);
    for (int j0 = 0; j0 < s.top_k; j0 += 32) {
      const int mine = lane_row(s, me.token, j0, rows);
      const A wmine = lane_weight(s, w, me.token, j0, mine);
      for (int j = 0; j < 32 && j0 + j < s.top_k; j += J) {
        P v[J][U];
        int row[J];
        A wj[J];
#pragma unroll
        for (int u = 0; u < J; ++u) {
          row[u] = __shfl_sync(kFull, mine, (j + u) & 31);   // lanes past top_k hold -1
          wj[u] = __shfl_sync(kFull, wmine, (j + u) & 31);
          const P* ph = (const P*)(h + (long long)row[u] * ldh) + c0;
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (row[u] >= 0 && c0 + k * s.lanes < s.pieces) v[u][k] = ph[k * s.lanes];
        }
#pragma unroll
        for (int u = 0; u < J; ++u) {
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if (row[u] < 0 || c0 + k * s.lanes >= s.pieces) continue;
            A f[N];
            v[u][k].up(f);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[k][i] += wj[u] * f[i];
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (c0 + k * s.lanes >= s.pieces) continue;
      P o;
      o.down(sum[k]);
      py[c0 + k * s.lanes] = o;
    }
  }
}

// The dot products of a token's pairs go over its whole row: all of the row's columns belong to
// one group of threads, J pairs at a time, and are summed in a fixed order (over a thread's
// pieces, over the lanes, over the warps).
template <typename T, int N>
__global__ void __launch_bounds__(kThreads, N * sizeof(T) == 16 ? 4 : sizeof(T) == 8 ? 2 : 3)
    combine_grad_kernel(Shape s, const T* __restrict__ dy, int ldy, const T* __restrict__ h,
                        int ldh, int rows, const typename Value<T>::Acc* __restrict__ w,
                        T* __restrict__ dh, int lddh, typename Value<T>::Acc* __restrict__ dw) {
  using A = typename Value<T>::Acc;
  using P = Pack<T, N>;
  constexpr int J = 4;
  constexpr int U = combine_pieces(N * sizeof(T));
  __shared__ A part[kThreads / 32][J];
  const Place me = place(s);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = s.lanes / 32, first = warp / warps * warps;
  const long long token = me.token < 0 ? 0 : me.token;
  const P* py = (const P*)(dy + token * ldy);
  for (int j0 = 0; j0 < s.top_k; j0 += J) {
    int row[J];
    A wj[J], dot[J];
#pragma unroll
    for (int u = 0; u < J; ++u) {
      const long long p = token * s.top_k + j0 + u;
      row[u] = me.token >= 0 && j0 + u < s.top_k ? s.pair_row[p] : -1;
      if (row[u] >= rows) row[u] = -1;
      wj[u] = w && row[u] >= 0 ? w[p] : A(1);
      dot[u] = A(0);
    }
    if (me.token >= 0) {
      for (long long c = me.at; c < s.pieces; c += (long long)s.lanes * U) {
        P g[U], v[J][U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (c + k * s.lanes < s.pieces) g[k] = py[c + k * s.lanes];
#pragma unroll
        for (int u = 0; u < J; ++u) {
          const P* ph = (const P*)(h + (long long)row[u] * ldh) + c;
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (dw && row[u] >= 0 && c + k * s.lanes < s.pieces) v[u][k] = ph[k * s.lanes];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (c + k * s.lanes >= s.pieces) continue;
          A gf[N];
          g[k].up(gf);
#pragma unroll
          for (int u = 0; u < J; ++u) {
            if (row[u] < 0) continue;
            A f[N];
            if (dw) {
              v[u][k].up(f);
#pragma unroll
              for (int i = 0; i < N; ++i) dot[u] += gf[i] * f[i];
            }
            if (dh) {
#pragma unroll
              for (int i = 0; i < N; ++i) f[i] = wj[u] * gf[i];
              P o;
              o.down(f);
              ((P*)(dh + (long long)row[u] * lddh))[c + k * s.lanes] = o;
            }
          }
        }
      }
    }
    if (!dw) continue;
#pragma unroll
    for (int u = 0; u < J; ++u) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[u] += __shfl_xor_sync(kFull, dot[u], o);
      if (lane == 0) part[warp][u] = dot[u];
    }
    __syncthreads();
    if (me.token >= 0 && me.at < J && j0 + me.at < s.top_k) {
      A sum = A(0);
      for (int k = 0; k < warps; ++k) sum += part[first + k][me.at];
      dw[token * s.top_k + j0 + me.at] = sum;
    }
    __syncthreads();
  }
}

// The largest of 16, 8, 4 (and 2) bytes on which all rows of a matrix start.
int grain(const DenseView& m, int bytes) {
  const unsigned long long all = (uintptr_t)m.data | (unsigned long long)(m.ld * bytes);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// As many threads per token as its pieces keep busy, `each` per thread.
Shape shape_for(const RoutesView& r, int pieces, int each) {
  Shape s{r.pair_row, r.tokens, r.top_k, pieces, 32};
  while (s.lanes < kThreads && (long long)s.lanes * each < pieces) s.lanes *= 2;
  return s;
}

dim3 grid_for(const Shape& s, long long per_cta_pieces) {
  const int per = kThreads / s.lanes;
  const long long y = ((long long)s.pieces + per_cta_pieces - 1) / per_cta_pieces;
  return dim3((unsigned)(((long long)s.tokens + per - 1) / per), (unsigned)(y > 65535 ? 65535 : y));
}

template <typename T, typename F>
void by_pieces(long long cols, int grain, F&& f) {
  constexpr int n16 = 16 / sizeof(T), n8 = 8 / sizeof(T), n4 = 4 / sizeof(T);
  if (grain >= 16 && cols % n16 == 0) return f(T(), std::integral_constant<int, n16>());
  if constexpr (sizeof(T) == 4)
    if (grain >= 8 && cols % n8 == 0) return f(T(), std::integral_constant<int, n8>());
  if constexpr (sizeof(T) == 2)
    if (grain >= 4 && cols % n4 == 0) return f(T(), std::integral_constant<int, n4>());
  return f(T(), std::integral_constant<int, 1>());
}

// f(T{}, N): N elements per piece, the most that every row starts and ends on.
template <typename F>
void by_type(int type, long long cols, int grain, F&& f) {
  switch (type) {
    case kF64: return by_pieces<double>(cols, grain, f);
    case kF32: return by_pieces<float>(cols, grain, f);
    case kF16: return by_pieces<__half>(cols, grain, f);
    default: return by_pieces<__nv_bfloat16>(cols, grain, f);
  }
}

int bytes_of(int type) { return type == kF64 ? 8 : type == kF32 ? 4 : 2; }

}  // namespace

int launch_dispatch(const RoutesView& r, const DenseView& x, const void* w, const DenseView& y,
                    cudaStream_t s) {
  if (r.tokens == 0 || x.cols == 0 || y.rows == 0) return 0;
  const int b = bytes_of(x.type);
  by_type(x.type, x.cols, std::min(grain(x, b), grain(y, b)), [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    const Shape sh = shape_for(r, (int)(x.cols / N), dispatch_pieces(N * sizeof(T)));
    launch(nullptr, dispatch_kernel<T, N>, grid_for(sh, sh.lanes * dispatch_pieces(N * sizeof(T))),
           kThreads, 0, s, 1, sh, (const T*)x.data, x.ld,
           (const typename Value<T>::Acc*)w, (T*)y.data, y.ld, y.rows);
  });
  return 1;
}

int launch_combine(const RoutesView& r, const DenseView& h, const void* w, const DenseView& y,
                   cudaStream_t s) {
  if (r.tokens == 0 || y.cols == 0) return 0;
  const int b = bytes_of(h.type);
  by_type(h.type, h.cols, std::min(grain(h, b), grain(y, b)), [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int N = decltype(n)::value;
    const Shape sh = shape_for(r, (int)(h.cols / N), combine_pieces(N * sizeof(T)));
    launch(nullptr, combine_kernel<T, N>, grid_for(sh, sh.lanes * combine_pieces(N * sizeof(T))),
           kThreads, 0, s, 1, sh, (const T*)h.data, h.ld, h.rows,
           (const typename Value<T>::Acc*)w, (T*)y.data, y.ld);
  });
  return 1;
}

int launch_combine_grad(const RoutesView& r, const DenseView& dy, const DenseView* h, const void* w,
                        const DenseView* dh, void* dw, cudaStream_t s) {
  if (r.tokens == 0 || (dy.cols == 0 && !dw)) return 0;
  const int b = bytes_of(dy.type);
  const int g = std::min({grain(dy, b), h ? grain(*h, b) : 16, dh ? grain(*dh, b) : 16});
  by_type(dy.type, dy.cols, g, [&](auto t, auto n) {
    using T = decltype(t);
    using A = typename Value<T>::Acc;
    constexpr int N = decltype(n)::value;
    const Shape sh = shape_for(r, (int)(dy.cols / N), combine_pieces(N * sizeof(T)));
    const int per = kThreads / sh.lanes;
    launch(nullptr, combine_grad_kernel<T, N>, (unsigned)((r.tokens + per - 1ll) / per), kThreads,
           0, s, 1, sh, (const T*)dy.data, dy.ld, h ? (const T*)h->data : nullptr, h ? h->ld : 0,
           h ? h->rows : dh->rows, (const A*)w, dh ? (T*)dh->data : nullptr, dh ? dh->ld : 0,
           (A*)dw);
  });
  return 1;
}

}  // namespace appt
