// Internal interface of the routed products (include/appt_spgemm.h): checked arguments from
// experts.cu to the kernels' launchers. Every launcher is asynchronous on its stream and returns
// the number of kernels it launched.
#pragma once
#include <cuda_runtime.h>
#include <atomic>
#include <cstddef>
#include <cstdint>

namespace appt {

struct LaunchFailed {   // thrown by launch(), turned into a status at the C entry
  cudaError_t error;
};

// As launch()'s cluster: no clusters, and the kernel may start before the stream's kernel before
// it has ended (it waits for that end itself, before it reads what that kernel writes or writes
// what it reads).
constexpr int kAfterStart = 0;

// kernel<<<grid, block, smem, s>>>(args...) in clusters of `cluster` CTAs, with the launch's own
// status (an error that an earlier call of the program left behind is not taken for it). The opt-in
// to more than 48 KB of shared memory, static and dynamic together, is per device and kept in
// *opted, a bit per device.
constexpr size_t kStaticMost = 16 * 1024;   // of any kernel here that also has dynamic memory
template <typename... P, typename... A>
void launch(std::atomic<unsigned long long>* opted, void (*kernel)(P...), dim3 grid, dim3 block,
            size_t smem, cudaStream_t s, int cluster, A... args) {
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024 - kStaticMost) {
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(opted->load() >> dev & 1)) {
      int most = 0;
      e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
      cudaFuncAttributes fa = {};
      if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kernel);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 most - (int)fa.sharedSizeBytes);
      if (e == cudaSuccess) opted->fetch_or(1ull << dev);
    }
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    if (cluster == kAfterStart) {
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
    } else {
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = cluster;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = cluster != 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw LaunchFailed{e};
  }
}

enum DenseType : int { kF64 = 0, kF32 = 1, kF16 = 2, kBF16 = 3, kE4M3 = 4, kI32 = 5, kI64 = 6 };

constexpr int kMaxExperts = 1024;
constexpr int kScaleBlock = 128;   // columns (and rows of weights) that share a scale

struct DenseView {        // row-major, ld in elements
  void* data = nullptr;
  long long rows = 0, cols = 0, ld = 0;
  int type = kF32;
};

struct RoutesView {
  const int* pair_row = nullptr;
  int tokens = 0, top_k = 0;
};

struct ScaledView {
  DenseView q;
  float* scale = nullptr;
  long long scale_ld = 0;
};

struct BlocksView {
  const void* data = nullptr;
  const float* scale = nullptr;
  long long groups = 0, rows = 0, cols = 0, ld = 0, group_stride = 0;
};

// route.cu
size_t route_workspace_bytes(long long pairs, int experts);
int launch_route(const DenseView& ids, int experts, int* expert_ptr, int* row_pair, int* pair_row,
                 int* counts, cudaStream_t s);
// routed_rows.cu
int launch_dispatch(const RoutesView& r, const DenseView& x, const void* w, const DenseView& y,
                    cudaStream_t s);
int launch_combine(const RoutesView& r, const DenseView& h, const void* w, const DenseView& y,
                   cudaStream_t s);
int launch_combine_grad(const RoutesView& r, const DenseView& dy, const DenseView* h, const void* w,
                        const DenseView* dh, void* dw, cudaStream_t s);
// quantize.cu
int launch_quantize(const DenseView& x, bool gated, const int* rows_ptr, const RoutesView* routes,
                    const ScaledView& q, cudaStream_t s);
// scaled_product.cu
int launch_scaled_product(const ScaledView& a, const BlocksView& w, const int* group_ptr,
                          const DenseView& y, int sms, cudaStream_t s);
// The tile of Y that a product of these sizes goes by: fewer than 128 rows with the weights as lanes.
struct ProductTile {
  int rows, cols;
};
ProductTile scaled_product_tile(long long rows, long long n, long long groups, int sms);
// Makes later products give up (or not).
void scaled_product_give_up(bool on);
// Reads and clears the current device's record of products that gave up a wait (a cudaError_t).
int scaled_product_status(int* gave_up);

}  // namespace appt
