// Products of rows in 8 bits with each group's matrix in 8 bits, scales by blocks of 128:
//
//   Y[r, n] = sum_b sa[b, r] sw[g, n / 128, b] sum_{k in block b} a[r, k] w[g, n, k]
//
// for the rows r of group g (a block-diagonal product; one group is the dense one). The scales
// change along the sum, so the tensor cores form one block's products at a time (four
// instructions of 32 columns) in tensor memory, and two warpgroups scale each partial tile and
// add it to fp32 sums in registers while the next block's products run.
//
// Roles (12 warps): 0 loads tiles by TMA into a ring; 1 issues the products, each block into the
// next of the tensor-memory buffers; 2 and 3 copy the block's scales to a ring of their own; 4..11
// read a buffer (each warpgroup half of its columns), scale and add, and write Y at the end of a
// tile. CTAs are persistent and take tiles in turn, the tiles of a group's columns next to each
// other.
//
// Two layouts. With many rows per group the rows are the 128 lanes of a tile and the weights its
// columns: a thread owns a row, its scale is one register. With few rows per group the weights
// are the lanes and the rows the columns (16 to 64 of them): a tile of 128 rows would be mostly
// padding, and the tensor cores' time goes by the columns. A row's scale is then one per column,
// read from shared memory.
// With fewer tiles than half the SMs, a cluster of CTAs splits a tile along K and adds its parts
// through distributed shared memory in the order of the ranks, so the result does not depend on
// timing.
#include <cuda.h>
#include <cuda_runtime.h>
#include <mutex>
#include "common.cuh"
#include "experts.h"
#include "tcgen05.cuh"
#include "values.cuh"

namespace appt {

using namespace sm100;

// Set by a kernel that gave up a wait; read and cleared by scaled_product_status.
__device__ int g_product_gave_up;

namespace {

constexpr int kThreads = 384;
constexpr int kLanes = 128;                 // rows of a tile's first operand
constexpr int kTileBytes = kLanes * kScaleBlock;
constexpr int kScaleStages = 8;
constexpr int kMaxStages = 10;
constexpr int kMaxBuffers = 4;
constexpr int kSharedMax = 227 * 1024;

struct Params {
  const float* sa;
  long long sa_ld;
  const float* sw;
  const int* group_ptr;
  void* y;
  long long ldy;
  int rows, n, k_blocks, n_blocks, groups, type;
  bool vec;            // rows of y start on 16 bytes
};

// Tables of the groups, filled at the start of a kernel.
struct Groups {
  int tile[kMaxExperts + 1];   // first tile of a group (tiles along rows)
  int row[kMaxExperts + 1];    // first row; a group ends where the next one begins
};

struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t tfull[kMaxBuffers], tempty[kMaxBuffers];
  uint64_t sfull[kScaleStages], sempty[kScaleStages];
  uint64_t drain;
};

template <bool kSwap, int kCols>
struct Shape {
  static constexpr int kStageBytes = kTileBytes + kCols * kScaleBlock;
  static constexpr int kRowTile = kSwap ? kCols : kLanes;      // rows of Y per tile
  static constexpr int kNTile = kSwap ? kLanes : kCols;        // columns of Y per tile
  static constexpr int kWScales = (kNTile + kScaleBlock - 1) / kScaleBlock;
  static constexpr int kScaleFloats = kRowTile + 4;            // rows, then up to 2 of the weights
  static constexpr int kBuffers = 512 / kCols < kMaxBuffers ? 512 / kCols : kMaxBuffers;
  // 128 sums a thread: the adding warps take registers of the other four. 128 x 56 + 256 x 216 =
  // 62,464 of the 384 x 168 = 64,512 that the launch holds.
  static constexpr bool kMoveRegs = kCols == 256;
  static constexpr int kTmemColumns = kBuffers * kCols < 32 ? 32 : kBuffers * kCols;
  static constexpr int kFixedBytes = (int)sizeof(Groups) + (int)sizeof(Barriers) + 64 +
                                     kScaleStages * kScaleFloats * 4 + 1024;
  static constexpr int kStages = (kSharedMax - kFixedBytes) / kStageBytes < kMaxStages
                                     ? (kSharedMax - kFixedBytes) / kStageBytes
                                     : kMaxStages;
  static constexpr int kBytes = kStages * kStageBytes + kFixedBytes;
};

__device__ __forceinline__ void store_one(const Params& p, long long at, float v) {
  if (p.type == kF32) ((float*)p.y)[at] = v;
  else if (p.type == kF16) ((__half*)p.y)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)p.y)[at] = __float2bfloat16_rn(v);
}

// 8 neighbouring values of a row
__device__ __forceinline__ void store_eight(const Params& p, long long at, const float* v) {
  if (p.type == kF32) {
    float4* d = (float4*)((float*)p.y + at);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if (p.type == kF16) {
    Pack<__half, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = __float2half_rn(v[i]);
    *(Pack<__half, 8>*)((__half*)p.y + at) = o;
  } else {
    Pack<__nv_bfloat16, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = __float2bfloat16_rn(v[i]);
    *(Pack<__nv_bfloat16, 8>*)((__nv_bfloat16*)p.y + at) = o;
  }
}

// Fills the tables: a group begins at the largest of the offsets so far, cut to the rows, so that
// groups never overlap and never leave the operands, whatever the offsets are.
template <int kRowTile>
__device__ void fill_groups(const Params& p, Groups* t) {
  for (int g = threadIdx.x; g <= p.groups; g += kThreads)
    t->row[g] = p.group_ptr ? min(max(p.group_ptr[g], 0), p.rows) : (g ? p.rows : 0);
  __syncthreads();
  if (threadIdx.x < 32) {
    int most = 0, tiles = 0;
    for (int g0 = 0; g0 <= p.groups; g0 += 32) {
      const int g = g0 + threadIdx.x;
      int r = g <= p.groups ? t->row[g] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, r, o);
        if ((int)threadIdx.x >= o) r = max(r, v);
      }
      r = max(r, most);
      // tiles of the group before: rows from its begin (the lane below) to r
      int prev = __shfl_up_sync(kFull, r, 1);
      if (threadIdx.x == 0) prev = g0 ? most : r;
      const int mine = (r - prev + kRowTile - 1) / kRowTile;
      const int incl = tiles + warp_incl_scan(mine);
      if (g <= p.groups) {
        t->row[g] = r;
        t->tile[g] = incl;
      }
      most = __shfl_sync(kFull, r, 31);
      tiles = __shfl_sync(kFull, incl, 31);
    }
  }
  __syncthreads();
}

struct Tile {
  int group, row, row_end, n;    // first row, end of the group's rows, first column of Y
};

template <int kRowTile, int kNTile>
__device__ __forceinline__ Tile tile_at(const Params& p, const Groups* t, long long i,
                                        int n_tiles) {
  const int rt = (int)(i / n_tiles);
  int lo = 0, hi = p.groups - 1;   // the last group whose first tile is <= rt
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t->tile[mid] <= rt) lo = mid; else hi = mid - 1;
  }
  return Tile{lo, t->row[lo] + (rt - t->tile[lo]) * kRowTile, t->row[lo + 1],
              (int)(i % n_tiles) * kNTile};
}

template <bool kSwap, int kCols>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ CUtensorMap map_w, const Params p, int splits) {
  using S = Shape<kSwap, kCols>;
  constexpr int kHalf = kCols / 2;            // columns of a warpgroup
  constexpr int kChunk = kHalf < 32 ? kHalf : 32;
  extern __shared__ char raw[];
  char* base = (char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  Groups* groups = (Groups*)(base + S::kStages * S::kStageBytes);
  float* scales = (float*)(groups + 1);
  Barriers* bars = (Barriers*)(((uintptr_t)(scales + kScaleStages * S::kScaleFloats) + 7) &
                               ~(uintptr_t)7);
  uint32_t* tmem_slot = (uint32_t*)(bars + 1);
  volatile int* gave_up = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(smem_u32(&bars->full[i]), 1);
      mbar_init(smem_u32(&bars->empty[i]), 1);
    }
    for (int i = 0; i < S::kBuffers; ++i) {
      mbar_init(smem_u32(&bars->tfull[i]), 1);
      mbar_init(smem_u32(&bars->tempty[i]), 8);
    }
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(smem_u32(&bars->sfull[i]), 64);
      mbar_init(smem_u32(&bars->sempty[i]), 8);
    }
    mbar_init(smem_u32(&bars->drain), 1);
    mbar_init_fence();
    *gave_up = 0;
    tma_prefetch_map(&map_a);
    tma_prefetch_map(&map_w);
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), S::kTmemColumns);
  fence_before();
  fill_groups<S::kRowTile>(p, groups);   // ends with a barrier of the CTA
  fence_after();
  const uint32_t tmem = *tmem_slot;

  const int n_tiles = (p.n + S::kNTile - 1) / S::kNTile;
  const long long tiles = (long long)groups->tile[p.groups] * n_tiles;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const long long first = blockIdx.x / splits, step = gridDim.x / splits;
  const int kb0 = (int)((long long)p.k_blocks * rank / splits);
  const int kb1 = (int)((long long)p.k_blocks * (rank + 1) / splits);

  if (warp < 4) {
    if (S::kMoveRegs) regs_fewer<56>();
    if (warp == 0 && lane == 0) {
      // ---- tiles by TMA
      int it = 0;
      bool ok = true;
      for (long long i = first; ok && i < tiles; i += step) {
        const Tile t = tile_at<S::kRowTile, S::kNTile>(p, groups, i, n_tiles);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % S::kStages;
          ok = mbar_wait(smem_u32(&bars->empty[st]), (it / S::kStages & 1) ^ 1, gave_up);
          if (!ok) break;
          const uint32_t full = smem_u32(&bars->full[st]);
          const uint32_t at = smem_u32(base + st * S::kStageBytes);
          mbar_expect(full, S::kStageBytes);
          tma_load_2d(kSwap ? at + kTileBytes : at, &map_a, kb * kScaleBlock, t.row, full);
          tma_load_3d(kSwap ? at : at + kTileBytes, &map_w, kb * kScaleBlock, t.n, t.group, full);
        }
      }
      if (!ok)   // let the loads in flight land before the CTA ends
        for (int j = max(0, it - S::kStages); j < it; ++j)
          for (int n = 0; n < kWaitTries; ++n)
            if (mbar_try(smem_u32(&bars->full[j % S::kStages]), j / S::kStages & 1)) break;
    } else if (warp == 1 && lane == 0) {
      // ---- products
      constexpr uint32_t idesc = instr_desc(kLanes, kCols);
      int it = 0;
      bool ok = true;
      for (long long i = first; ok && i < tiles; i += step) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % S::kStages, b = it % S::kBuffers;
          ok = mbar_wait(smem_u32(&bars->full[st]), it / S::kStages & 1, gave_up) &&
               mbar_wait(smem_u32(&bars->tempty[b]), (it / S::kBuffers & 1) ^ 1, gave_up);
          if (!ok) break;
          fence_after();
          const uint32_t at = smem_u32(base + st * S::kStageBytes);
          const uint64_t da = smem_desc(at), db = smem_desc(at + kTileBytes);
#pragma unroll
          for (int k = 0; k < kScaleBlock / 32; ++k)
            mma_f8(tmem + b * kCols, da + 2 * k, db + 2 * k, idesc, k > 0);
          mma_commit(smem_u32(&bars->empty[st]));
          mma_commit(smem_u32(&bars->tfull[b]));
        }
      }
      // products (and their arrivals) in flight end before the CTA does
      mma_commit(smem_u32(&bars->drain));
      for (int n = 0; n < kWaitTries; ++n)
        if (mbar_try(smem_u32(&bars->drain), 0)) break;
    } else if (warp >= 2) {
      // ---- scales
      const int me = threadIdx.x - 64;
      int it = 0;
      bool ok = true;
      for (long long i = first; ok && i < tiles; i += step) {
        const Tile t = tile_at<S::kRowTile, S::kNTile>(p, groups, i, n_tiles);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % kScaleStages;
          ok = mbar_wait(smem_u32(&bars->sempty[st]), (it / kScaleStages & 1) ^ 1, gave_up);
          if (!ok) break;
          float* s = scales + st * S::kScaleFloats;
          for (int r = me; r < S::kRowTile; r += 64) {
            const bool in = t.row + r < t.row_end;
            cp_async_4(smem_u32(s + r), p.sa + kb * p.sa_ld + (in ? t.row + r : t.row), in);
          }
          if (me < S::kWScales) {
            const int nb = t.n / kScaleBlock + me;
            const bool in = nb < p.n_blocks;
            cp_async_4(smem_u32(s + S::kRowTile + me),
                       p.sw + ((long long)t.group * p.n_blocks + (in ? nb : 0)) * p.k_blocks + kb,
                       in);
          }
          cp_async_arrive(smem_u32(&bars->sfull[st]));
        }
      }
      cp_async_wait_all();
    }
    __syncwarp();
  } else {
    // ---- scaling, adding, writing
    if (S::kMoveRegs) regs_more<216>();
    const int wg = (warp - 4) / 4, quarter = warp & 3;
    const int who = quarter * 32 + lane;         // lane of the tile
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16) + wg * kHalf;
    int it = 0;
    bool ok = true;
    for (long long i = first; ok && i < tiles; i += step) {
      const Tile t = tile_at<S::kRowTile, S::kNTile>(p, groups, i, n_tiles);
      float sum[kHalf];
#pragma unroll
      for (int c = 0; c < kHalf; ++c) sum[c] = 0.f;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % kScaleStages, b = it % S::kBuffers;
        ok = mbar_wait(smem_u32(&bars->sfull[st]), it / kScaleStages & 1, gave_up) &&
             mbar_wait(smem_u32(&bars->tfull[b]), it / S::kBuffers & 1, gave_up);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        const float* s = scales + st * S::kScaleFloats;
        const float sw = s[S::kRowTile + (S::kWScales > 1 ? wg : 0)];
        const float scale = kSwap ? sw : sw * s[who];
        fence_after();
        uint32_t part[2][kChunk];
        tmem_load(part[0], mine + b * kCols);
#pragma unroll
        for (int c = 0; c < kHalf; c += kChunk) {
          uint32_t(&now)[kChunk] = part[c / kChunk & 1];
          tmem_wait(now);
          if (c + kChunk < kHalf)
            tmem_load(part[(c / kChunk & 1) ^ 1], mine + b * kCols + c + kChunk);
          else {
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->tempty[b]));
          }
#pragma unroll
          for (int j = 0; j < kChunk; ++j) {
            const float f = kSwap ? scale * s[wg * kHalf + c + j] : scale;
            sum[c + j] = fmaf(__uint_as_float(now[j]), f, sum[c + j]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->sempty[st]));
      }
      if (!ok) break;
      if constexpr (kSwap) {
        if (splits > 1) {
          // the stages are free: every load has been used by a product that is done
          float* part = (float*)base;
#pragma unroll
          for (int c = 0; c < kHalf; ++c) part[(wg * kHalf + c) * kLanes + who] = sum[c];
        } else if (t.n + who < p.n) {
#pragma unroll
          for (int c = 0; c < kHalf; ++c) {
            const int r = t.row + wg * kHalf + c;
            if (r < t.row_end) store_one(p, r * p.ldy + t.n + who, sum[c]);
          }
        }
      } else {
        const int r = t.row + who;
        if (r < t.row_end) {
          const long long at = r * p.ldy + t.n + wg * kHalf;
#pragma unroll
          for (int c = 0; c < kHalf; c += 8) {
            const int n = t.n + wg * kHalf + c;
            if (p.vec && n + 8 <= p.n) {
              store_eight(p, at + c, &sum[c]);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < p.n) store_one(p, at + c + j, sum[c + j]);
            }
          }
        }
      }
    }
    if (!ok && lane == 0) g_product_gave_up = 1;
  }
  if constexpr (kSwap) {
    if (splits > 1) {
      // one tile per cluster: every CTA adds its share of the columns over all ranks
      cluster_sync();
      if (first < tiles && warp >= 4) {
        const Tile t = tile_at<S::kRowTile, S::kNTile>(p, groups, first, n_tiles);
        const int who = threadIdx.x & (kLanes - 1), wg = (warp - 4) / 4;
        for (int c = rank + splits * wg; c < kCols; c += 2 * splits) {
          const int r = t.row + c;
          if (r >= t.row_end || t.n + who >= p.n) continue;
          const uint32_t at = smem_u32((float*)base + c * kLanes + who);
          float v = 0.f;
          for (int q = 0; q < splits; ++q) v += load_cluster(map_shared(at, q));
          store_one(p, r * p.ldy + t.n + who, v);
        }
      }
      cluster_sync();   // no CTA leaves while another reads its part
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem, S::kTmemColumns);
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static std::atomic<void*> cached{nullptr};
  void* fn = cached.load();
  if (!fn) {
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000,
                                                           cudaEnableDefault, &found);
    if (e != cudaSuccess || found != cudaDriverEntryPointSuccess || !fn)
      throw LaunchFailed{e == cudaSuccess ? cudaErrorSymbolNotFound : e};
    cached.store(fn);
  }
  return (EncodeTiled)fn;
}

// Boxes of `box` rows x 128 bytes, swizzled; columns and rows outside the matrix read as zeros.
CUtensorMap map_of(const void* data, long long cols, long long rows, long long ld,
                   long long groups, long long group_stride, int box, int dims) {
  CUtensorMap m;
  const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t stride[2] = {(cuuint64_t)ld, (cuuint64_t)group_stride};
  const cuuint32_t boxes[3] = {kScaleBlock, (cuuint32_t)box, 1}, ones[3] = {1, 1, 1};
  if (encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(data), size, stride,
                     boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    throw LaunchFailed{cudaErrorInvalidValue};
  return m;
}

template <bool kSwap, int kCols>
void product(const ScaledView& a, const BlocksView& w, const Params& p, int sms, cudaStream_t s) {
  using S = Shape<kSwap, kCols>;
  static_assert(S::kStages >= 3, "");
  static_assert(!kSwap || kCols * kLanes * 4 <= S::kStages * S::kStageBytes, "");
  static std::atomic<unsigned long long> opted{0};
  const CUtensorMap ma = map_of(a.q.data, a.q.cols, a.q.rows, a.q.ld, 1, 0, S::kRowTile, 2);
  const CUtensorMap mw =
      map_of(w.data, w.cols, w.rows, w.ld, w.groups, w.group_stride, S::kNTile, 3);
  // the most tiles that the groups' sizes allow
  const long long n_tiles = (p.n + S::kNTile - 1) / S::kNTile;
  const long long row_tiles =
      p.rows / S::kRowTile + (w.groups < p.rows ? w.groups : (long long)p.rows);
  const long long tiles = row_tiles * n_tiles;
  int splits = 1;
  if (kSwap)
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= p.k_blocks) splits *= 2;
  const long long ctas = splits > 1 ? tiles * splits : tiles < sms ? tiles : sms;
  launch(&opted, product_kernel<kSwap, kCols>, dim3((unsigned)ctas), dim3(kThreads), S::kBytes, s,
         splits, ma, mw, p, splits);
}

}  // namespace

int launch_scaled_product(const ScaledView& a, const BlocksView& w, const int* group_ptr,
                          const DenseView& y, int sms, cudaStream_t s) {
  Params p;
  p.sa = a.scale;
  p.sa_ld = a.scale_ld;
  p.sw = w.scale;
  p.group_ptr = group_ptr;
  p.y = y.data;
  p.ldy = y.ld;
  p.rows = (int)y.rows;
  p.n = (int)w.rows;
  p.k_blocks = (int)((w.cols + kScaleBlock - 1) / kScaleBlock);
  p.n_blocks = (int)((w.rows + kScaleBlock - 1) / kScaleBlock);
  p.groups = (int)w.groups;
  p.type = y.type;
  const int b = y.type == kF32 ? 4 : 2;
  p.vec = (uintptr_t)y.data % 16 == 0 && y.ld * b % 16 == 0;
  const long long each = (y.rows + w.groups - 1) / w.groups;   // rows per group, if all are used
  if (each <= 16) product<true, 16>(a, w, p, sms, s);
  else if (each <= 32) product<true, 32>(a, w, p, sms, s);
  else if (each <= 64) product<true, 64>(a, w, p, sms, s);
  else if (w.rows <= 128) product<false, 128>(a, w, p, sms, s);
  else product<false, 256>(a, w, p, sms, s);
  return 1;
}

int scaled_product_status(int* gave_up) {
  cudaError_t e = cudaMemcpyFromSymbol(gave_up, g_product_gave_up, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && *gave_up)
    e = cudaMemcpyToSymbol(g_product_gave_up, &zero, sizeof(int));
  return e;
}

}  // namespace appt
