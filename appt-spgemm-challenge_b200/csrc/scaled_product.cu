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
// next of the tensor-memory buffers; 2 and 3 copy the block's scales to a ring of their own where
// they are needed by column; 4..11 read a buffer (each warpgroup half of its columns), scale and
// add, and write Y at the end of a tile. CTAs are persistent and take tiles in turn, the tiles of a
// group's columns next to each other.
//
// Two layouts. With many rows per group the rows are the 128 lanes of a tile and the weights its
// columns: a thread owns a row, its scale is one register. With few rows per group the weights
// are the lanes and the rows the columns (16 to 64 of them): a tile of 128 rows would be mostly
// padding, and the tensor cores' time goes by the columns. A row's scale is then one per column,
// read from shared memory.
// With fewer tiles than half the SMs, a cluster of CTAs splits a tile along K. Each CTA sends its
// sums through distributed shared memory to the columns' owners, which add them in the order of
// the ranks, so the result does not depend on timing.
//
// Many rows: no unit is full (tensor pipe 55 %, issue slots 44 %, DRAM 8 %); the adding warps' chain
// sets the time. A block of 128 x 256 takes the tensor cores 512 cycles and the adding warps some
// 820: 256 for its fused multiply-adds, about as much for the reads of tensor memory between them,
// which do not overlap, the rest for waiting on one buffer and handing back the other. Neither more
// adding warps (4 warpgroups of 64 columns), nor pairs of CTAs on tiles of 256 rows (a third less
// traffic from L2), nor halves of 128 columns with barriers of their own were faster. 8192 x 8192 x
// 4096 takes 259 us, 2.1 PFLOP/s (300 us at the clocks that 1000 W leave it), 32,768 sorted rows x
// 2048 x 2048 over 64 groups 174 us. Few rows: bound by the weights' bytes; 128 rows over 56 of 64
// groups, 4096 x 2048, 78 us, 6.1 TB/s; one row x 4096 x 4096 6.2 us.
#include <cuda.h>
#include <cuda_runtime.h>
#include <climits>
#include "common.cuh"
#include "experts.h"
#include "tcgen05.cuh"
#include "values.cuh"

namespace appt {

using namespace sm100;

// Set by a kernel that gave up a wait; read and cleared by scaled_product_status.
__device__ int g_product_gave_up;

namespace {

constexpr int kLanes = 128;                 // rows of a tile's first operand
constexpr int kTileBytes = kLanes * kScaleBlock;
constexpr int kScaleStages = 8;
constexpr int kMaxStages = 10;
constexpr int kMaxBuffers = 4;
constexpr int kSharedMax = 227 * 1024;
constexpr int kOutBox = 32 * 128;
constexpr int kRegsFew = 72, kRegsMany = 216;   // see Shape::kMoveRegs

struct Params {
  const float* sa;
  long long sa_ld;
  const float* sw;
  const int* group_ptr;
  void* y;
  long long ldy;
  int rows, n, k_blocks, n_blocks, groups, type;
  int n_tiles;               // tiles of a row of tiles
  int step_rows, step_cols;  // from a CTA's tile to its next
  int splits_log2;           // CTAs that share a tile's K
  bool give_up;        // asked to, after a tile's first block (before its only one)
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
  static constexpr int kScaleFloats = kSwap ? kCols + 4 : 0;   // the rows', then the weights'
  static constexpr int kBuffers = 512 / kCols < kMaxBuffers ? 512 / kCols : kMaxBuffers;
  // 128 sums a thread: the adding warps take registers of the other four. 128 x 72 + 256 x 216 =
  // 64,512, the 384 x 168 that the launch holds.
  static constexpr bool kMoveRegs = kCols == 256;
  static constexpr int kTmemColumns = kBuffers * kCols < 32 ? 32 : kBuffers * kCols;
  static constexpr int kGroups = 2;                            // adding warpgroups
  static constexpr int kThreads = 128 + 128 * kGroups;
  static constexpr int kPart = kCols / kGroups;                // columns of a warpgroup
  // Y on its way out: a warp's boxes of 32 rows x 128 bytes, enough for its 16-bit values
  static constexpr int kOutBoxes = kPart / 64;
  static constexpr int kOutBytes =
      kSwap ? kCols * kLanes * 4 : 4 * kGroups * kOutBoxes * kOutBox;
  static constexpr int kFixedBytes = kOutBytes + (int)sizeof(Groups) + (int)sizeof(Barriers) + 64 +
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

// The first `rows` rows and `left_cols` columns of a warp's boxes to Y; not inlined, for it would
// take registers that the sums need.
template <typename T, int kBoxes>
__device__ __noinline__ void store_boxes(T* y, long long ldy, bool vec, const char* boxes, int rows,
                                         int left_cols) {
  constexpr int kPer = 16 / sizeof(T), kPieces = 8 * kBoxes;
  const int lane = threadIdx.x & 31, cols = min(left_cols, kPieces * kPer);
  auto piece = [&](int r, int j) {
    return (const T*)(boxes + j / 8 * kOutBox + r * 128 + ((j % 8) ^ (r & 7)) * 16);
  };
  if (vec) {
    const int j = lane % kPieces, left = cols - j * kPer;
#pragma unroll 4
    for (int r = lane / kPieces; r < rows; r += 32 / kPieces) {
      T* to = y + r * ldy + j * kPer;
      if (left >= kPer) *(uint4*)to = *(const uint4*)piece(r, j);
      else
        for (int i = 0; i < left; ++i) to[i] = piece(r, j)[i];
    }
  } else {
    for (int c = lane; c < cols; c += 32) {
#pragma unroll 8
      for (int r = 0; r < rows; ++r) y[r * ldy + c] = piece(r, c / kPer)[c % kPer];
    }
  }
}

// A warp's 32 rows x N columns of Y, a row per thread, through boxes in shared memory that TMA
// copies while the warp goes on with its next tile. The 16-byte pieces of a row change places by
// the row (the 128-byte swizzle), which spreads the threads over the banks. Stores from registers
// are 16 bytes of 32 rows at a time and took 4,500 cycles a tile, this takes a quarter.
// A group's last rows, rows that TMA cannot address, and columns of which the last 16 bytes are not
// all Y's (TMA would write the whole piece) are stored from the boxes instead.
template <typename T, int N, int kBoxes>
__device__ __forceinline__ void write_rows(const Params& p, const CUtensorMap* map, char* boxes,
                                           const uint64_t* v, int row, int rows, int n) {
  constexpr int kPer = 16 / sizeof(T), kCols = 128 / sizeof(T);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c0 = 0; c0 < N; c0 += kBoxes * kCols) {   // once, or twice for 32 bits
    bulk_wait_read();                                // the copies before these (the issuer's)
    __syncwarp();
#pragma unroll
    for (int c = c0; c < c0 + kBoxes * kCols; c += kPer) {
      char* box = boxes + (c - c0) / kCols * kOutBox;
      float f[kPer];
#pragma unroll
      for (int i = 0; i < kPer; i += 2) untwo(v[(c + i) / 2], f[i], f[i + 1]);
      Pack<T, kPer> o;
      o.down(f);
      *(Pack<T, kPer>*)(box + lane * 128 + ((c % kCols) / kPer ^ (lane & 7)) * 16) = o;
    }
    if (p.vec && rows >= 32 && (p.n % kPer == 0 || n + c0 + kBoxes * kCols <= p.n)) {
      bulk_fence();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int b = 0; b < kBoxes; ++b)
          tma_store_2d(map, n + c0 + b * kCols, row, smem_u32(boxes + b * kOutBox));
        bulk_commit();
      }
    } else {
      __syncwarp();
      store_boxes<T, kBoxes>((T*)p.y + (long long)row * p.ldy + n + c0, p.ldy, p.vec, boxes,
                             min(rows, 32), p.n - n - c0);
    }
  }
}

// Fills the tables: a group begins at the largest of the offsets so far, cut to the rows, so that
// groups never overlap and never leave the operands, whatever the offsets are.
template <int kRowTile>
__device__ void fill_groups(const Params& p, Groups* t) {
  if (!p.group_ptr) {
    if (threadIdx.x == 0) {
      t->row[0] = t->tile[0] = 0;
      t->row[1] = p.rows;
      t->tile[1] = (p.rows + kRowTile - 1) / kRowTile;
    }
    __syncthreads();
    return;
  }
  for (int g = threadIdx.x; g <= p.groups; g += blockDim.x)
    t->row[g] = min(max(p.group_ptr[g], 0), p.rows);
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

// A CTA's tiles, in order: index i, i + step, ... in rows of n_tiles tiles.
template <int kRowTile, int kNTile>
struct Tiles {
  const Groups* t;
  int rows, n_tiles, step_rows, step_cols, row, col, group;
  __device__ __forceinline__ Tiles(const Params& p, const Groups* groups, int i)
      : t(groups), rows(groups->tile[p.groups]), n_tiles(p.n_tiles), step_rows(p.step_rows),
        step_cols(p.step_cols) {
    row = i / n_tiles;
    col = i - row * n_tiles;
    group = 0;
  }
  __device__ __forceinline__ bool more() const { return row < rows; }
  __device__ __forceinline__ Tile at() {
    while (t->tile[group + 1] <= row) ++group;   // ends: row is below the last entry
    return Tile{group, t->row[group] + (row - t->tile[group]) * kRowTile, t->row[group + 1],
                col * kNTile};
  }
  __device__ __forceinline__ void next() {
    row += step_rows;
    col += step_cols;
    if (col >= n_tiles) col -= n_tiles, ++row;
  }
};

template <bool kSwap, int kCols>
__global__ void __launch_bounds__(Shape<kSwap, kCols>::kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_y, const Params p) {
  using S = Shape<kSwap, kCols>;
  constexpr int kPart = S::kPart;             // columns of a warpgroup
  extern __shared__ char raw[];
  char* base = (char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  char* out = base + S::kStages * S::kStageBytes;   // on 1024 bytes, as the swizzle wants it
  float* shares = (float*)out;                      // partial sums of a tile whose K is split
  Groups* groups = (Groups*)(out + S::kOutBytes);
  float* scales = (float*)(groups + 1);
  Barriers* bars = (Barriers*)(((uintptr_t)(scales + kScaleStages * S::kScaleFloats) + 7) &
                               ~(uintptr_t)7);
  uint32_t* tmem_slot = (uint32_t*)(bars + 1);
  volatile int* gave_up = (volatile int*)(tmem_slot + 1);

  const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane < S::kStages) {
      mbar_init(smem_u32(&bars->full[lane]), 1);
      mbar_init(smem_u32(&bars->empty[lane]), 1);
    }
    if (lane < S::kBuffers) {
      mbar_init(smem_u32(&bars->tfull[lane]), 1);
      mbar_init(smem_u32(&bars->tempty[lane]), 4 * S::kGroups);
    }
    if (lane < kScaleStages) {
      mbar_init(smem_u32(&bars->sfull[lane]), 64);
      mbar_init(smem_u32(&bars->sempty[lane]), 8);
    }
    if (lane == 0) {
      mbar_init(smem_u32(&bars->drain), 1);
      *gave_up = 0;
      tma_prefetch_map(&map_a);
      tma_prefetch_map(&map_w);
    }
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), S::kTmemColumns);
  fence_before();
  fill_groups<S::kRowTile>(p, groups);   // ends with a barrier of the CTA
  fence_after();
  const uint32_t tmem = *tmem_slot;

  const int splits = 1 << p.splits_log2;
  const int rank = kSwap && splits > 1 ? (int)cluster_rank() : 0;
  // Every thread arrives here and waits once: warps that write to the other CTAs' shared memory
  // before they do (the CTAs run by then), the others at the end of their roles.
  if (kSwap && splits > 1) cluster_arrive();
  Tiles<S::kRowTile, S::kNTile> order(p, groups, blockIdx.x >> p.splits_log2);
  const int kb0 = p.k_blocks * rank >> p.splits_log2;   // k_blocks < 2^24
  const int kb1 = p.k_blocks * (rank + 1) >> p.splits_log2;

  if (warp < 4) {
    if (S::kMoveRegs) regs_fewer<kRegsFew>();
    if (warp == 0) {
      // ---- tiles by TMA
      int it = 0, st = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (; ok && order.more(); order.next()) {
        const Tile t = order.at();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          ok = mbar_wait(smem_u32(&bars->empty[st]), phase, gave_up);
          if (!ok) break;
          const uint32_t full = smem_u32(&bars->full[st]);
          const uint32_t at = smem_u32(base + st * S::kStageBytes);
          if (elect_one()) {
            mbar_expect(full, S::kStageBytes);
            tma_load_2d(kSwap ? at + kTileBytes : at, &map_a, kb * kScaleBlock, t.row, full);
            tma_load_3d(kSwap ? at : at + kTileBytes, &map_w, kb * kScaleBlock, t.n, t.group, full);
          }
          if (++st == S::kStages) st = 0, phase ^= 1;
        }
      }
      // Loads in flight land before the CTA ends: there are some where another role has given up.
      for (int j = max(0, it - S::kStages); j < it; ++j)
        mbar_drain(smem_u32(&bars->full[j % S::kStages]), j / S::kStages & 1);
    } else if (warp == 1) {
      // ---- products
      constexpr uint32_t idesc = instr_desc(kLanes, kCols);
      int st = 0, b = 0;
      uint32_t phase = 0, bphase = 1;
      bool ok = true;
      const int last = p.give_up ? min(kb0 + 1, kb1 - 1) : kb1;
      for (; ok && order.more(); order.next()) {
        for (int kb = kb0; kb < last; ++kb) {
          ok = mbar_wait(smem_u32(&bars->full[st]), phase, gave_up) &&
               mbar_wait(smem_u32(&bars->tempty[b]), bphase, gave_up);
          if (!ok) break;
          fence_after();
          const uint32_t at = smem_u32(base + st * S::kStageBytes);
          const uint64_t da = smem_desc(at), db = smem_desc(at + kTileBytes);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kScaleBlock / 32; ++k)
              mma_f8(tmem + b * kCols, da + 2 * k, db + 2 * k, idesc, k > 0);
            mma_commit(smem_u32(&bars->tfull[b]));
            mma_commit(smem_u32(&bars->empty[st]));
          }
          __syncwarp();
          if (++st == S::kStages) st = 0, phase ^= 1;
          if (++b == S::kBuffers) b = 0, bphase ^= 1;
        }
        if (last < kb1) {
          *gave_up = 1;
          ok = false;
        }
      }
      // products (and their arrivals) in flight end before the CTA does
      if (elect_one()) mma_commit(smem_u32(&bars->drain));
      __syncwarp();
      mbar_drain(smem_u32(&bars->drain), 0);
    } else if (kSwap) {
      // ---- scales
      const int me = threadIdx.x - 64;
      int it = 0;
      bool ok = true;
      for (; ok && order.more(); order.next()) {
        const Tile t = order.at();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % kScaleStages;
          ok = mbar_wait(smem_u32(&bars->sempty[st]), (it / kScaleStages & 1) ^ 1, gave_up);
          if (!ok) break;
          float* s = scales + st * S::kScaleFloats;
          for (int r = me; r < S::kRowTile; r += 64) {
            const bool in = t.row + r < t.row_end;
            cp_async_4(smem_u32(s + r), p.sa + kb * p.sa_ld + (in ? t.row + r : t.row), in);
          }
          if (me == 0)
            cp_async_4(smem_u32(s + S::kRowTile),
                       p.sw + ((long long)t.group * p.n_blocks + t.n / kScaleBlock) * p.k_blocks + kb,
                       true);
          cp_async_arrive(smem_u32(&bars->sfull[st]));
        }
      }
      cp_async_wait_all();
    }
    __syncwarp();
    if (kSwap && splits > 1) cluster_wait();
  } else {
    // ---- scaling, adding, writing
    if (S::kMoveRegs) regs_more<kRegsMany>();
    const int wg = (warp - 4) / 4, quarter = warp & 3;
    const int who = quarter * 32 + lane;         // lane of the tile
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16) + wg * kPart;
    int it = 0;
    bool ok = true;
    uint64_t pairs[kPart / 2];   // sums of neighbouring columns
    auto full_bar = [&](int n) { return smem_u32(&bars->tfull[n % S::kBuffers]); };
    auto full_phase = [&](int n) { return (uint32_t)(n / S::kBuffers & 1); };
    auto buffer = [&](int n) { return mine + n % S::kBuffers * kCols; };
    auto buffer_read = [&](int n) {
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed(smem_u32(&bars->tempty[n % S::kBuffers]));
    };
    auto clear = [&] {
#pragma unroll
      for (int c = 0; c < kPart / 2; ++c) pairs[c] = 0;
    };
    // What a warp that gave up has not computed leaves as NaN, this tile and the CTA's next ones.
    auto incomplete = [&] {
#pragma unroll
      for (int c = 0; c < kPart / 2; ++c) pairs[c] = ~0ull;
    };
    if constexpr (!kSwap) {
      // A thread's scales come two blocks ahead, those of its next tile before it writes this one.
      const float *pa, *pw;
      float a0, w0, a1, w1;
      auto begin = [&](const Tile& t) {
        pa = p.sa + min(t.row + who, t.row_end - 1);
        pw = p.sw + ((long long)t.group * p.n_blocks +
                     min((t.n + wg * kPart) / kScaleBlock, p.n_blocks - 1)) * p.k_blocks;
        const int second = min(1, p.k_blocks - 1), third = min(2, p.k_blocks - 1);
        a0 = pa[0], w0 = pw[0];
        a1 = pa[second * p.sa_ld], w1 = pw[second];
        pa += third * p.sa_ld, pw += third;   // the next block's but one, or the last again
      };
      // Adds one partial tile, kChunk columns at a time, and hands its buffer back as soon as the
      // last of them is in registers.
      constexpr int kChunk = 16;
      // (no copy from one pair of scales to the other: it would wait for a load in flight)
      auto block = [&](float& a, float& w, int kb) {
        ok = mbar_wait(full_bar(it), full_phase(it), gave_up);
        if (!ok) return;
        fence_after();
        const uint64_t scale = two(a * w, a * w);
#pragma unroll
        for (int c = 0; c < kPart; c += kChunk) {
          uint32_t now[kChunk];
          tmem_load(now, buffer(it) + c);
          if (c == 0) {
            a = *pa, w = *pw;
            if (kb + 3 < p.k_blocks) pa += p.sa_ld, ++pw;
          }
          tmem_wait(now);
          if (c + kChunk == kPart) buffer_read(it);
#pragma unroll
          for (int j = 0; j < kChunk; j += 2)
            pairs[(c + j) / 2] = fma_two(now[j], now[j + 1], scale, pairs[(c + j) / 2]);
        }
        ++it;
      };
      Tile t = {};
      if (order.more()) begin(t = order.at());
      while (order.more()) {
        clear();
        for (int kb = 0; ok && kb < p.k_blocks; kb += 2) {
          block(a0, w0, kb);
          if (ok && kb + 1 < p.k_blocks) block(a1, w1, kb + 1);
        }
        if (!ok) incomplete();
        const Tile done = t;
        order.next();
        if (order.more()) begin(t = order.at());
        const int row = done.row + quarter * 32, rows = done.row_end - row, n = done.n + wg * kPart;
        if (rows <= 0 || n >= p.n) continue;
        char* boxes = out + (warp - 4) * S::kOutBoxes * kOutBox;
        if (p.type == kF32)
          write_rows<float, kPart, S::kOutBoxes>(p, &map_y, boxes, pairs, row, rows, n);
        else if (p.type == kF16)
          write_rows<__half, kPart, S::kOutBoxes>(p, &map_y, boxes, pairs, row, rows, n);
        else
          write_rows<__nv_bfloat16, kPart, S::kOutBoxes>(p, &map_y, boxes, pairs, row, rows, n);
      }
      bulk_wait();
    } else {
      bool waited = false;
      for (; order.more(); order.next()) {
        const Tile t = order.at();
        clear();
        for (int kb = kb0; ok && kb < kb1; ++kb, ++it) {
          const int st = it % kScaleStages;
          ok = mbar_wait(smem_u32(&bars->sfull[st]), it / kScaleStages & 1, gave_up);
          if (!ok) break;
          const float* s = scales + st * S::kScaleFloats;
          const float sw = s[S::kRowTile];
          ok = mbar_wait(full_bar(it), full_phase(it), gave_up);
          if (!ok) break;
          fence_after();
          uint32_t now[kPart];
          tmem_load(now, buffer(it));
          tmem_wait(now);
          buffer_read(it);
#pragma unroll
          for (int c = 0; c < kPart; c += 2)
            pairs[c / 2] = fma_two(now[c], now[c + 1],
                                   two(sw * s[wg * kPart + c], sw * s[wg * kPart + c + 1]),
                                   pairs[c / 2]);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars->sempty[st]));
        }
        if (!ok) incomplete();
        float sum[kPart];
#pragma unroll
        for (int c = 0; c < kPart; c += 2) untwo(pairs[c / 2], sum[c], sum[c + 1]);
        if (splits > 1) {
          // every rank gets its share of the columns from all: c % splits == rank
          cluster_wait();
          waited = true;
#pragma unroll
          for (int c = 0; c < kPart; ++c) {
            const int col = wg * kPart + c;
            if (t.row + col < t.row_end)
              store_cluster(map_shared(smem_u32(shares + ((rank * kCols + col) >> p.splits_log2) *
                                                             kLanes + who),
                                       col & (splits - 1)),
                            sum[c]);
          }
        } else if (t.n + who < p.n) {
#pragma unroll
          for (int c = 0; c < kPart; ++c) {
            const int r = t.row + wg * kPart + c;
            if (r < t.row_end) store_one(p, r * p.ldy + t.n + who, sum[c]);
          }
        }
      }
      if (splits > 1 && !waited) cluster_wait();
    }
    if (!ok && lane == 0) g_product_gave_up = 1;
    __syncwarp();
  }
  if constexpr (kSwap) {
    if (splits > 1) {
      // one tile per cluster: every CTA adds its share of the columns over all ranks, in their order
      cluster_sync();
      Tiles<S::kRowTile, S::kNTile> mine(p, groups, blockIdx.x >> p.splits_log2);
      if (mine.more() && warp >= 4) {
        const Tile t = mine.at();
        const int who = threadIdx.x & (kLanes - 1), wg = (warp - 4) / 4;
        const int each = kCols >> p.splits_log2;
        const int last = t.n + who < p.n ? t.row_end - t.row : 0;
        for (int i = wg; i < each && i * splits + rank < last; i += 2) {
          float sum = 0.f;
          for (int q = 0; q < splits; ++q) sum += shares[(q * each + i) * kLanes + who];
          store_one(p, (t.row + i * splits + rank) * p.ldy + t.n + who, sum);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem, S::kTmemColumns);
  }
}

std::atomic<bool> g_give_up{false};

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

// Boxes of `box` rows x 128 bytes, swizzled, of elements of `bytes`; columns and rows outside the
// matrix read as zeros. Strides are in bytes.
CUtensorMap map_of(const void* data, long long cols, long long rows, long long ld,
                   long long groups, long long group_stride, int box, int dims, int bytes = 1) {
  CUtensorMap m;
  const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t stride[2] = {(cuuint64_t)ld, (cuuint64_t)group_stride};
  const cuuint32_t boxes[3] = {128u / bytes, (cuuint32_t)box, 1}, ones[3] = {1, 1, 1};
  const CUtensorMapDataType type = bytes == 4   ? CU_TENSOR_MAP_DATA_TYPE_UINT32
                                   : bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  if (encode_tiled()(&m, type, dims, const_cast<void*>(data), size, stride,
                     boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    throw LaunchFailed{cudaErrorInvalidValue};
  return m;
}

// The most tiles along the rows that groups of any sizes can have (one group's size is known).
long long row_tiles_for(long long rows, long long groups, int tile) {
  if (groups == 1) return (rows + tile - 1) / tile;
  return rows / tile + (groups < rows ? groups : rows);
}

template <bool kSwap, int kCols>
void product(const ScaledView& a, const BlocksView& w, Params p, int sms, cudaStream_t s) {
  using S = Shape<kSwap, kCols>;
  static_assert(S::kStages >= 3, "");
  static std::atomic<unsigned long long> opted{0};
  if (S::kMoveRegs) {
    // a kernel built to fewer registers could never hand the adding warps theirs: they would wait
    static std::atomic<int> regs{0};
    if (regs.load() == 0) {
      cudaFuncAttributes fa = {};
      const cudaError_t e = cudaFuncGetAttributes(&fa, product_kernel<kSwap, kCols>);
      if (e != cudaSuccess) throw LaunchFailed{e};
      regs.store(fa.numRegs);
    }
    if (regs.load() * S::kThreads < 128 * kRegsFew + 256 * kRegsMany)
      throw LaunchFailed{cudaErrorLaunchOutOfResources};
  }
  const CUtensorMap ma = map_of(a.q.data, a.q.cols, a.q.rows, a.q.ld, 1, 0, S::kRowTile, 2);
  const CUtensorMap mw =
      map_of(w.data, w.cols, w.rows, w.ld, w.groups, w.group_stride, S::kNTile, 3);
  CUtensorMap my = ma;   // (of Y only where its rows allow one)
  if (!kSwap && p.vec) {
    const int b = p.type == kF32 ? 4 : 2;
    my = map_of(p.y, p.n, p.rows, p.ldy * b, 1, 0, 32, 2, b);
  }
  const long long n_tiles = (p.n + S::kNTile - 1) / S::kNTile;
  const long long tiles = row_tiles_for(p.rows, p.groups, S::kRowTile) * n_tiles;
  if (tiles > INT_MAX - sms) throw LaunchFailed{cudaErrorInvalidValue};   // no memory holds such a Y
  int log2 = 0;
  if (kSwap)
    // (a cluster's CTAs share a GPC, whose SMs the clusters may not all fill: a second wave of
    // them took 13.7 us where 7 was expected)
    while (log2 < 3 && tiles << (log2 + 1) <= sms * 7 / 8 && 2 << log2 <= p.k_blocks) ++log2;
  const long long step = log2 || tiles < sms ? tiles : sms;
  p.n_tiles = (int)n_tiles;
  p.step_rows = (int)(step / n_tiles);
  p.step_cols = (int)(step % n_tiles);
  p.splits_log2 = log2;
  launch(&opted, product_kernel<kSwap, kCols>, dim3((unsigned)(step << log2)), dim3(S::kThreads),
         S::kBytes, s, 1 << log2, ma, mw, my, p);
}

}  // namespace

// Few rows per group: the weights as lanes, and as few columns as mostly hold a group's rows (half
// as many again as the mean; one group's rows are known). Else the rows as lanes, unless that
// leaves more than half of the SMs without a tile, where the other layout can split K. 256 columns
// unless 128 fill the SMs so much better that the narrower tile's waves, four fifths as long, are
// fewer in time. Measured, in us, as 16 | 32 | 64 columns of rows | 128 | 256 columns of weights:
//   64 groups, 2048 x 2048:  8 rows each  50 | 50 | 53 | 58 |  53
//                           16 rows each  54 | 50 | 54 | 61 |  56
//                           48 rows each 120 | 79 | 57 | 63 |  57
//                          128 rows each 276 |169 |125 | 84 |  73
//   one group,  4096 x 4096:  48 rows      13 | 12 | 10 | 15 |  19
//                            512 rows      68 | 44 | 29 | 17 |  21
//                           1024 rows     130 | 73 | 52 | 29 |  22
//   one group,  512 x 2048:  128 rows       9 |  7 |  7 | 10 |  13
ProductTile scaled_product_tile(long long rows, long long n, long long groups, int sms) {
  const long long fits = groups == 1 ? rows : rows * 3 / 2 / groups;
  const long long row_tiles = row_tiles_for(rows, groups, kLanes);
  const long long narrow = row_tiles * ((n + 127) / 128), wide = row_tiles * ((n + 255) / 256);
  auto waves = [&](long long tiles) { return (tiles + sms - 1) / sms; };
  if (fits <= 16) return {16, kLanes};
  if (fits <= 32) return {32, kLanes};
  if (fits <= 64 || narrow * 2 <= sms) return {64, kLanes};
  return {kLanes, waves(wide) * 5 > waves(narrow) * 4 ? 128 : 256};
}

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
  p.give_up = g_give_up.load(std::memory_order_relaxed);
  const int b = y.type == kF32 ? 4 : 2;
  p.vec = (uintptr_t)y.data % 16 == 0 && y.ld * b % 16 == 0;
  const ProductTile tile = scaled_product_tile(p.rows, p.n, p.groups, sms);
  if (tile.rows == 16) product<true, 16>(a, w, p, sms, s);
  else if (tile.rows == 32) product<true, 32>(a, w, p, sms, s);
  else if (tile.rows == 64) product<true, 64>(a, w, p, sms, s);
  else if (tile.cols == 128) product<false, 128>(a, w, p, sms, s);
  else product<false, 256>(a, w, p, sms, s);
  return 1;
}

void scaled_product_give_up(bool on) { g_give_up.store(on, std::memory_order_relaxed); }

int scaled_product_status(int* gave_up) {
  cudaError_t e = cudaMemcpyFromSymbol(gave_up, g_product_gave_up, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && *gave_up)
    e = cudaMemcpyToSymbol(g_product_gave_up, &zero, sizeof(int));
  return e;
}

}  // namespace appt
