// Sorting (token, expert) pairs by expert: a stable counting sort.
//
//   expert_ptr[e] = number of kept pairs with an id below e
//   row of pair p = expert_ptr[id] + number of kept pairs before p with the same id
//
// The pairs are cut into one contiguous chunk per CTA. An expert's base in chunk b is expert_ptr[e]
// plus its counts in the chunks before b, so a CTA needs the other chunks' counts and no order
// among CTAs. Up to 8 chunks are one cluster and read each other's counts from shared memory; more
// get them from a kernel that counts first (whose end the placing kernel waits for only once its
// own counting is done). Within a chunk each warp owns a contiguous part, counts it per expert in
// shared memory, and places 32 pairs at a time: the rank among equal ids of the 32 lanes is a
// popcount of the match mask. No atomic decides an order, so equal inputs give equal outputs.
//
// Bound by latency: a chain of some six barriers and two trips to memory. 256 pairs (64 experts)
// 2.9 us, 4,096 (256 experts) 5.0 us, 524,288 (6.2 MB) 10.9 us, of which the counting kernel takes
// 4 and a quarter of the rest is the match.
#include <cuda_runtime.h>
#include "common.cuh"
#include "experts.h"
#include "tcgen05.cuh"

namespace appt {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;           // steps of 32 pairs that a warp has in flight
constexpr int kChunkMin = 512;      // pairs per CTA: below, more CTAs do not pay
constexpr int kClusterChunks = 8;   // the largest portable cluster
constexpr int kClusterPairs = 8 * 2048;
constexpr int kMaxChunks = 128;

// 1, 2, 4 or 8 chunks where one cluster does it in a single launch, or any number above. 16,384
// pairs of 256 experts take 6.9 us as a cluster and 6.8 us counted first, but a launch more on the
// host; 65,536 take 7.0 us counted first and would take 12 as a cluster.
int chunks_for(long long pairs) {
  const long long n = (pairs + kChunkMin - 1) / kChunkMin;
  if (pairs > kClusterPairs) return n > kMaxChunks ? kMaxChunks : (int)n;
  return n > 4 ? 8 : n > 2 ? 4 : n > 1 ? 2 : 1;
}

// How a CTA learns the other chunks' counts.
enum Others { kNone, kCluster, kCounted };

__device__ __forceinline__ void wait_for_grid_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_grid_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// kPacked: a token's ids follow the token's before without a gap (no division then).
template <typename IdType, bool kPacked>
struct Ids {
  using Id = IdType;
  const Id* data;
  long long ld;
  int top_k, experts, pairs;
  // the pair's expert, or -1 for an id outside [0, experts)
  __device__ __forceinline__ int at(int p) const {
    const Id e = data[kPacked ? p : (long long)(p / top_k) * ld + p % top_k];
    return e >= 0 && e < (Id)experts ? (int)e : -1;
  }
};

template <typename I>
__global__ void __launch_bounds__(kThreads) route_count_kernel(I ids, int chunk, int* counts) {
  extern __shared__ int hist[];
  let_next_grid_start();
  for (int e = threadIdx.x; e < ids.experts; e += kThreads) hist[e] = 0;
  __syncthreads();
  const long long lo = (long long)blockIdx.x * chunk;
  const long long hi = min(lo + chunk, (long long)ids.pairs);
#pragma unroll 4
  for (long long p = lo + threadIdx.x; p < hi; p += kThreads) {
    const int e = ids.at((int)p);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ids.experts; e += kThreads)
    counts[blockIdx.x * ids.experts + e] = hist[e];
}

// One warp's part of a chunk, [lo, hi), and how many warps have one.
__device__ __forceinline__ int warp_part(long long clo, long long chi, long long* lo,
                                         long long* hi) {
  const int n = chi > clo ? (int)(chi - clo) : 0;
  const int part = max(((n + kWarps - 1) / kWarps + 31) / 32 * 32, 32);
  *lo = min(clo + (long long)part * (threadIdx.x >> 5), chi);
  *hi = min(*lo + part, chi);
  return (n + part - 1) / part;
}

// (One CTA per SM is asked for: left to itself the compiler stays at 32 registers, its loads wait
// for each other, and the largest case takes 18 us instead of 11.)
template <typename I, Others kOthers>
__global__ void __launch_bounds__(kThreads, 1)
    route_place_kernel(I ids, int chunk, const int* __restrict__ counts, int* expert_ptr,
                       int* row_pair, int* pair_row) {
  extern __shared__ int next[];   // [kWarps][experts]: first counts, then the next row to give
  __shared__ long long scan[kWarps + 1];
  __shared__ int mine_of[kMaxExperts], total_of[kMaxExperts], before_of[kMaxExperts];
  const int experts = ids.experts, lane = threadIdx.x & 31;
  int* mine = next + (threadIdx.x >> 5) * experts;
  long long lo, hi;
  const long long clo = (long long)blockIdx.x * chunk;
  const int warps = warp_part(clo, min(clo + chunk, (long long)ids.pairs), &lo, &hi);
  for (int i = threadIdx.x; i < warps * experts; i += kThreads) next[i] = 0;
  __syncthreads();
  int id[kBatch];   // 32 pairs each, on their way together
  auto fetch = [&](long long p0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const long long p = p0 + 32 * k + lane;
      id[k] = p < hi ? ids.at((int)p) : -1;
    }
  };
  for (long long p0 = lo; p0 < hi; p0 += 32 * kBatch) {
    fetch(p0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (id[k] >= 0) atomicAdd(&mine[id[k]], 1);
  }
  __syncthreads();
  const int e = threadIdx.x;   // experts <= kThreads
  int total = 0, before = 0;
  if (kOthers != kCounted && e < experts) {
#pragma unroll 8
    for (int w = 0; w < warps; ++w) total += next[w * experts + e];
  }
  if (kOthers == kCluster) {
    if (e < experts) mine_of[e] = total;
    sm100::cluster_sync();
    if (e < experts) {
      const uint32_t at = sm100::smem_u32(&mine_of[e]);
      total = 0;
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = __float_as_int(sm100::load_cluster(sm100::map_shared(at, b)));
        total += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
    }
    sm100::cluster_sync();   // no CTA leaves while another reads its counts
  }
  if (kOthers == kCounted) {
    // several threads per expert, each with every so-manyth chunk
    int wide = 32;
    while (wide < experts) wide *= 2;
    const int who = e % wide, part = e / wide, parts = kThreads / wide;
    if (e < experts) total_of[e] = before_of[e] = 0;
    __syncthreads();
    wait_for_grid_before();
    if (who < experts) {
#pragma unroll 16
      for (int b = part; b < (int)gridDim.x; b += parts) {
        const int c = __ldcg(&counts[b * experts + who]);
        total += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
      atomicAdd(&total_of[who], total);
      atomicAdd(&before_of[who], before);
    }
    __syncthreads();
    if (e < experts) {
      total = total_of[e];
      before = before_of[e];
    } else {
      total = 0;
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
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int c = next[w * experts + e];
      next[w * experts + e] = row;
      row += c;
    }
  }
  __syncthreads();
  for (long long p0 = lo; p0 < hi; p0 += 32 * kBatch) {
    if (hi - lo > 32 * kBatch) fetch(p0);   // else they are still here
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const long long p = p0 + 32 * k + lane;
      if (p0 + 32 * k >= hi) break;
      const unsigned same = __match_any_sync(kFull, id[k]);
      const int rank = __popc(same & lanemask_lt());
      int row = -1;
      if (id[k] >= 0) row = mine[id[k]] + rank;
      __syncwarp();
      if (id[k] >= 0 && rank == 0) mine[id[k]] += __popc(same);
      __syncwarp();
      if (p < hi) {
        pair_row[p] = row;
        if (row >= 0) row_pair[row] = (int)p;
      }
    }
  }
}

template <typename I>
int route(const DenseView& v, int experts, int* expert_ptr, int* row_pair, int* pair_row,
          int* counts, cudaStream_t s) {
  static std::atomic<unsigned long long> opted[3];
  const int pairs = (int)(v.rows * v.cols);
  const I ids{(const typename I::Id*)v.data, v.ld, (int)v.cols, experts, pairs};
  const int chunks = chunks_for(pairs);
  const int chunk = (int)(((long long)pairs + chunks - 1) / chunks);
  const size_t smem = kWarps * experts * sizeof(int);
  if (chunks == 1) {
    launch(&opted[0], route_place_kernel<I, kNone>, 1, kThreads, smem, s, 1, ids, chunk, nullptr,
           expert_ptr, row_pair, pair_row);
    return 1;
  }
  if (chunks <= kClusterChunks) {
    launch(&opted[1], route_place_kernel<I, kCluster>, chunks, kThreads, smem, s, chunks, ids,
           chunk, nullptr, expert_ptr, row_pair, pair_row);
    return 1;
  }
  launch(nullptr, route_count_kernel<I>, chunks, kThreads, experts * sizeof(int), s, 1, ids, chunk,
         counts);
  launch(&opted[2], route_place_kernel<I, kCounted>, chunks, kThreads, smem, s, kAfterStart, ids,
         chunk, counts, expert_ptr, row_pair, pair_row);
  return 2;
}

}  // namespace

size_t route_workspace_bytes(long long pairs, int experts) {
  const size_t n = (size_t)chunks_for(pairs) * experts * sizeof(int);
  return (n + 15) / 16 * 16;
}

int launch_route(const DenseView& ids, int experts, int* expert_ptr, int* row_pair, int* pair_row,
                 int* counts, cudaStream_t s) {
  const bool packed = ids.rows < 2 || ids.ld == ids.cols;
  auto go = [&](auto i) {
    return route<decltype(i)>(ids, experts, expert_ptr, row_pair, pair_row, counts, s);
  };
  if (ids.type == kI64) return packed ? go(Ids<long long, true>()) : go(Ids<long long, false>());
  return packed ? go(Ids<int, true>()) : go(Ids<int, false>());
}

}  // namespace appt
