// Sorting (token, expert) pairs by expert: a stable counting sort.
//
//   expert_ptr[e] = number of kept pairs with an id below e
//   row of pair p = expert_ptr[id] + number of kept pairs before p with the same id
//
// The pairs are cut into one contiguous chunk per CTA. With several chunks a first kernel counts
// each chunk's pairs per expert; the placing kernel then has every chunk's counts and needs no
// order among CTAs: an expert's base in chunk b is expert_ptr[e] plus its counts in chunks before
// b. Within a chunk each warp owns a contiguous part, counts it per expert in shared memory, and
// places 32 pairs at a time: the rank among equal ids of the 32 lanes is a popcount of the match
// mask. No atomic decides an order, so equal inputs give equal outputs.
#include <cuda_runtime.h>
#include "common.cuh"
#include "experts.h"

namespace appt {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kChunkMin = 4096;    // pairs per CTA below which more CTAs do not pay
constexpr int kMaxChunks = 128;

int chunks_for(long long pairs) {
  const long long n = (pairs + kChunkMin - 1) / kChunkMin;
  return n < 1 ? 1 : n > kMaxChunks ? kMaxChunks : (int)n;
}

template <typename Id>
struct Ids {
  const Id* data;
  long long ld;
  int top_k, experts, pairs;
  // the pair's expert, or -1 for an id outside [0, experts)
  __device__ __forceinline__ int at(int p) const {
    const long long i = ld == top_k ? p : (long long)(p / top_k) * ld + p % top_k;
    const Id e = data[i];
    return e >= 0 && e < (Id)experts ? (int)e : -1;
  }
};

template <typename Id>
__global__ void __launch_bounds__(kThreads) route_count_kernel(Ids<Id> ids, int chunk,
                                                               int* counts) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < ids.experts; e += kThreads) hist[e] = 0;
  __syncthreads();
  const long long lo = (long long)blockIdx.x * chunk;
  const long long hi = min(lo + chunk, (long long)ids.pairs);
  for (long long p = lo + threadIdx.x; p < hi; p += kThreads) {
    const int e = ids.at((int)p);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ids.experts; e += kThreads)
    counts[blockIdx.x * ids.experts + e] = hist[e];
}

// One warp's part of a chunk: [lo, hi).
__device__ __forceinline__ void warp_part(long long clo, long long chi, long long* lo,
                                          long long* hi) {
  const long long n = chi > clo ? chi - clo : 0;
  const long long part = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  *lo = min(clo + part * (threadIdx.x >> 5), chi);
  *hi = min(*lo + part, chi);
}

template <typename Id>
__global__ void __launch_bounds__(kThreads)
    route_place_kernel(Ids<Id> ids, int chunk, const int* __restrict__ counts, int* expert_ptr,
                       int* row_pair, int* pair_row) {
  extern __shared__ int next[];   // [kWarps][experts]: first counts, then the next row to give
  __shared__ long long scan[kWarps + 1];
  const int experts = ids.experts, lane = threadIdx.x & 31;
  int* mine = next + (threadIdx.x >> 5) * experts;
  for (int i = threadIdx.x; i < kWarps * experts; i += kThreads) next[i] = 0;
  __syncthreads();
  long long lo, hi;
  const long long clo = (long long)blockIdx.x * chunk;
  warp_part(clo, min(clo + chunk, (long long)ids.pairs), &lo, &hi);
  for (long long p = lo + lane; p < hi; p += 32) {
    const int e = ids.at((int)p);
    if (e >= 0) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  const int e = threadIdx.x;   // experts <= kThreads
  int total = 0, before = 0;
  if (e < experts) {
    if (gridDim.x == 1) {
      for (int w = 0; w < kWarps; ++w) total += next[w * experts + e];
    } else {
#pragma unroll 8
      for (int b = 0; b < gridDim.x; ++b) {
        const int c = counts[b * experts + e];
        total += c;
        before += b < blockIdx.x ? c : 0;
      }
    }
  }
  long long all;
  const int first = (int)block_excl_scan_ll<kThreads>(total, scan, &all);
  if (e < experts) {
    if (blockIdx.x == 0) {
      expert_ptr[e] = first;
      if (e == 0) expert_ptr[experts] = (int)all;
    }
    int row = first + before;
    for (int w = 0; w < kWarps; ++w) {
      const int c = next[w * experts + e];
      next[w * experts + e] = row;
      row += c;
    }
  }
  __syncthreads();
  for (long long p0 = lo; p0 < hi; p0 += 32) {
    const long long p = p0 + lane;
    const int id = p < hi ? ids.at((int)p) : -1;
    const unsigned same = __match_any_sync(kFull, id);
    const int rank = __popc(same & lanemask_lt());
    int row = -1;
    if (id >= 0) row = mine[id] + rank;
    __syncwarp();
    if (id >= 0 && rank == 0) mine[id] += __popc(same);
    __syncwarp();
    if (p < hi) {
      pair_row[p] = row;
      if (row >= 0) row_pair[row] = (int)p;
    }
  }
}

template <typename Id>
int route(const DenseView& v, int experts, int* expert_ptr, int* row_pair, int* pair_row,
          int* counts, cudaStream_t s) {
  static std::atomic<unsigned long long> opted{0};
  const int pairs = (int)(v.rows * v.cols);
  // a single row's ld is its own length
  const Ids<Id> ids{(const Id*)v.data, v.rows > 1 ? v.ld : v.cols, (int)v.cols, experts, pairs};
  const int chunks = chunks_for(pairs);
  const int chunk = (int)(((long long)pairs + chunks - 1) / chunks);
  if (chunks > 1)
    launch(nullptr, route_count_kernel<Id>, chunks, kThreads, experts * sizeof(int), s, 1, ids, chunk,
           counts);
  launch(&opted, route_place_kernel<Id>, chunks, kThreads, kWarps * experts * sizeof(int), s, 1, ids,
         chunk, counts, expert_ptr, row_pair, pair_row);
  return chunks > 1 ? 2 : 1;
}

}  // namespace

size_t route_workspace_bytes(long long pairs, int experts) {
  const size_t n = (size_t)chunks_for(pairs) * experts * sizeof(int);
  return (n + 15) / 16 * 16;
}

int launch_route(const DenseView& ids, int experts, int* expert_ptr, int* row_pair, int* pair_row,
                 int* counts, int sms, cudaStream_t s) {
  (void)sms;
  return ids.type == kI64 ? route<long long>(ids, experts, expert_ptr, row_pair, pair_row, counts, s)
                          : route<int>(ids, experts, expert_ptr, row_pair, pair_row, counts, s);
}

}  // namespace appt
