// Routed products: argument checks and the C entry points (include/appt_spgemm.h, "Routed
// products"). Sizes, pointers, alignment and overlap are checked before the first CUDA call, so a
// refused call has touched neither the device nor an output.
#include <cuda_runtime.h>
#include <atomic>
#include <climits>
#include <cstdint>
#include <exception>
#include <string>

#include "../../include/appt_spgemm.h"
#include "engine.h"
#include "experts.h"

namespace appt {
namespace {

struct Refused {   // thrown by the checks below, caught at the C entry
  int status;
  std::string what;
};

[[noreturn]] void refuse(const std::string& what, int status = kErrInvalid) {
  throw Refused{status, what};
}

void check_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver)
    refuse("no CUDA device", kErrNoDevice);
  refuse(std::string(what) + ": " + cudaGetErrorString(e), kErrCuda);
}

int type_bytes(int type) {
  switch (type) {
    case kF64: case kI64: return 8;
    case kF32: case kI32: return 4;
    case kF16: case kBF16: return 2;
    case kE4M3: return 1;
    default: return 0;
  }
}

// An address range with a row pitch, for the overlap and residency checks.
struct Span {
  const char* name;
  const char* p;
  long long rows, pitch, width;   // bytes
  bool out;
  long long bytes() const { return rows <= 0 || width <= 0 ? 0 : (rows - 1) * pitch + width; }
};

struct Spans {
  Span s[10];
  int n = 0;
  void add(const char* name, const void* p, long long rows, long long pitch, long long width,
           bool out) {
    s[n++] = Span{name, (const char*)p, rows, pitch, width, out};
  }
  void add(const char* name, const DenseView& m, bool out) {
    const long long b = type_bytes(m.type);
    add(name, m.data, m.rows, m.ld * b, m.cols * b, out);
  }
};

// Whether two strided ranges share a byte. Column ranges of one buffer (equal pitch) are told
// apart; anything else is compared by its whole extent.
bool overlap(const Span& a, const Span& b) {
  const long long na = a.bytes(), nb = b.bytes();
  if (!na || !nb || a.p + na <= b.p || b.p + nb <= a.p) return false;
  if (a.pitch == b.pitch && a.pitch > 0) {
    const long long p = a.pitch;
    const long long d = ((b.p - a.p) % p + p) % p;   // b's first column, seen from a's
    if (d >= a.width && d + b.width <= p) return false;
  }
  return true;
}

// Bytes that an operand may span: well above any memory, and no address arithmetic wraps below.
constexpr long long kLargest = 1ll << 50;

const DenseView view(const appt_dense* m, const char* name, unsigned types, int align = 0) {
  if (!m) refuse(std::string(name) + " is null");
  const int b = m->type < 0 || m->type > kI64 || !(types >> m->type & 1) ? 0 : type_bytes(m->type);
  if (!b) refuse(std::string(name) + ": type " + std::to_string(m->type) + " is not supported here");
  if (m->reserved != 0) refuse(std::string(name) + ": reserved is not 0");
  if (m->rows < 0 || m->rows >= INT_MAX || m->cols < 0 || m->cols >= INT_MAX)
    refuse(std::string(name) + ": rows and cols must lie in [0, 2^31 - 1)");
  DenseView v;
  v.rows = m->rows;
  v.cols = m->cols;
  v.type = m->type;
  v.ld = m->rows > 1 ? m->ld : (m->cols + 15) / 16 * 16;
  if (m->rows > 1 && (m->ld < m->cols || m->ld >= INT_MAX))
    refuse(std::string(name) + ": ld must be at least cols and below 2^31 - 1");
  if (v.ld > 0 && v.rows > kLargest / 8 / v.ld)
    refuse(std::string(name) + ": its rows reach further than any memory");
  v.data = m->data;
  if (v.rows > 0 && v.cols > 0) {
    if (!v.data) refuse(std::string(name) + ": null data");
    if ((uintptr_t)v.data % (align ? align : b))
      refuse(std::string(name) + ": data is not aligned to " + std::to_string(align ? align : b) +
             " bytes");
  }
  return v;
}

constexpr unsigned mask(int t) { return 1u << t; }
constexpr unsigned kValueTypes = mask(kF64) | mask(kF32) | mask(kF16) | mask(kBF16);
constexpr unsigned kShortTypes = mask(kF32) | mask(kF16) | mask(kBF16);

RoutesView view(const appt_routes* r, Spans* sp) {
  if (!r) refuse("routes is null");
  if (r->reserved != 0) refuse("routes: reserved is not 0");
  if (r->tokens < 0 || r->top_k < 1 || r->tokens >= INT_MAX ||
      r->tokens * (long long)r->top_k >= INT_MAX)
    refuse("routes: needs tokens >= 0, top_k >= 1 and tokens * top_k < 2^31 - 1");
  if (r->tokens > 0 && (!r->pair_row || (uintptr_t)r->pair_row % 4))
    refuse("routes: pair_row is null or not aligned to 4 bytes");
  RoutesView v;
  v.pair_row = r->pair_row;
  v.tokens = (int)r->tokens;
  v.top_k = r->top_k;
  const long long n = 4ll * v.tokens * v.top_k;
  sp->add("pair_row", v.pair_row, 1, n, n, false);
  return v;
}

ScaledView view(const appt_scaled* q, const char* name, bool out, int align, Spans* sp) {
  if (!q) refuse(std::string(name) + " is null");
  ScaledView v;
  v.q = view(&q->q, name, mask(kE4M3), align);
  v.scale = q->scale;
  v.scale_ld = q->scale_ld;
  const long long blocks = (v.q.cols + kScaleBlock - 1) / kScaleBlock;
  if (v.q.rows > 0 && v.q.cols > 0) {
    if (!v.scale || (uintptr_t)v.scale % 4)
      refuse(std::string(name) + ": scale is null or not aligned to 4 bytes");
    if (blocks > 1 && (v.scale_ld < v.q.rows || v.scale_ld >= INT_MAX))
      refuse(std::string(name) + ": scale_ld must be at least the rows and below 2^31 - 1");
  }
  if (blocks <= 1) v.scale_ld = v.q.rows;
  sp->add(name, v.q, out);
  sp->add("scale", v.scale, blocks, 4 * v.scale_ld, 4 * v.q.rows, out);
  return v;
}

void add_weights(const void* w, const char* name, const RoutesView& r, int type, bool out,
                 Spans* sp) {
  if (!w) return;
  const int b = type == kF64 ? 8 : 4;
  if ((uintptr_t)w % b)
    refuse(std::string(name) + " is not aligned to " + std::to_string(b) + " bytes");
  const long long n = (long long)b * r.tokens * r.top_k;
  sp->add(name, w, 1, n, n, out);
}

void check_overlap(const Spans& sp) {
  for (int i = 0; i < sp.n; ++i)
    for (int j = 0; j < sp.n; ++j)
      if (i != j && sp.s[i].out && (i < j || !sp.s[j].out) && overlap(sp.s[i], sp.s[j]))
        refuse(std::string(sp.s[i].name) + " overlaps " + sp.s[j].name);
}

// Makes `device` current for the call's lifetime and puts the caller's device back.
struct OnDevice {
  int before = -1;
  int sms = 0;
  explicit OnDevice(int device) {
    static std::atomic<int> count{-1};
    static std::atomic<int> sm_count[64];
    int n = count.load(std::memory_order_relaxed);
    if (n < 0) {
      check_cuda(cudaGetDeviceCount(&n), "cudaGetDeviceCount");
      count.store(n, std::memory_order_relaxed);
    }
    if (n == 0) refuse("no CUDA device", kErrNoDevice);
    if (device < 0 || device >= n || device >= 64) refuse("device ordinal out of range");
    int cur = 0;
    check_cuda(cudaGetDevice(&cur), "cudaGetDevice");
    if (cur != device) {
      check_cuda(cudaSetDevice(device), "cudaSetDevice");
      before = cur;
    }
    sms = sm_count[device].load(std::memory_order_relaxed);
    if (sms == 0) {
      check_cuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device),
                 "cudaDeviceGetAttribute");
      sm_count[device].store(sms, std::memory_order_relaxed);
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// Every buffer must be memory of `device`: a host pointer, or one of another device, would fault
// in the kernel.
void check_resident(const Spans& sp, int device) {
  for (int i = 0; i < sp.n; ++i) {
    if (!sp.s[i].bytes()) continue;
    cudaPointerAttributes a;
    check_cuda(cudaPointerGetAttributes(&a, sp.s[i].p), "cudaPointerGetAttributes");
    if (a.type == cudaMemoryTypeManaged) continue;
    if (a.type != cudaMemoryTypeDevice || a.device != device)
      refuse(std::string(sp.s[i].name) + " is not memory of device " + std::to_string(device));
  }
}

// Runs an entry's body; errors and exceptions become a status and appt_last_error().
template <typename F>
int guarded(const char* entry, F&& body) {
  try {
    body();
    return kOk;
  } catch (const Refused& r) {
    try {
      set_error(std::string(entry) + ": " + r.what);
    } catch (...) {
    }
    return r.status;
  } catch (const LaunchFailed& f) {
    try {
      set_error(std::string(entry) + ": launch failed: " + cudaGetErrorString(f.error));
    } catch (...) {
    }
    return kErrCuda;
  } catch (...) {   // out of host memory for a message
    return kErrOom;
  }
}

}  // namespace
}  // namespace appt

using namespace appt;

extern "C" {

size_t appt_route_workspace(int64_t tokens, int32_t top_k, int64_t experts) {
  if (tokens < 0 || tokens >= INT_MAX || top_k < 1 || tokens * (long long)top_k >= INT_MAX ||
      experts < 1 || experts > kMaxExperts)
    return 0;
  return route_workspace_bytes(tokens * (long long)top_k, (int)experts);
}

int appt_route(const appt_dense* ids, int64_t experts, int32_t* expert_ptr, int32_t* row_pair,
               int32_t* pair_row, void* workspace, size_t workspace_bytes, int32_t device,
               void* stream) {
  return guarded("appt_route", [&] {
    Spans sp;
    const DenseView v = view(ids, "ids", mask(kI32) | mask(kI64));
    if (v.cols < 1 || v.rows * v.cols >= INT_MAX)
      refuse("ids needs at least one column and fewer than 2^31 - 1 entries");
    if (experts < 1 || experts > kMaxExperts)
      refuse("experts must lie in [1, " + std::to_string(kMaxExperts) + "]");
    const long long pairs = v.rows * v.cols;
    if (!expert_ptr || (uintptr_t)expert_ptr % 4 ||
        (pairs && (!row_pair || !pair_row || (uintptr_t)row_pair % 4 || (uintptr_t)pair_row % 4)))
      refuse("a null output, or one not aligned to 4 bytes");
    const long long need = (long long)route_workspace_bytes(pairs, (int)experts);
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (size_t)need)
      refuse("workspace: needs " + std::to_string(need) + " bytes, aligned to 16");
    sp.add("ids", v, false);
    sp.add("expert_ptr", expert_ptr, 1, 4 * (experts + 1), 4 * (experts + 1), true);
    sp.add("row_pair", row_pair, 1, 4 * pairs, 4 * pairs, true);
    sp.add("pair_row", pair_row, 1, 4 * pairs, 4 * pairs, true);
    sp.add("workspace", workspace, 1, need, need, true);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_route(v, (int)experts, expert_ptr, row_pair, pair_row, (int*)workspace,
                               (cudaStream_t)stream));
  });
}

int appt_dispatch(const appt_routes* routes, const appt_dense* X, const void* weights,
                  const appt_dense* Y, int32_t device, void* stream) {
  return guarded("appt_dispatch", [&] {
    Spans sp;
    const RoutesView r = view(routes, &sp);
    const DenseView x = view(X, "X", kValueTypes), y = view(Y, "Y", kValueTypes);
    if (x.rows != r.tokens) refuse("X must have a row for each token");
    if (x.cols != y.cols || x.type != y.type) refuse("X and Y differ in columns or type");
    sp.add("X", x, false);
    sp.add("Y", y, true);
    add_weights(weights, "weights", r, x.type, false, &sp);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_dispatch(r, x, weights, y, (cudaStream_t)stream));
  });
}

int appt_combine(const appt_routes* routes, const appt_dense* H, const void* weights,
                 const appt_dense* Y, int32_t device, void* stream) {
  return guarded("appt_combine", [&] {
    Spans sp;
    const RoutesView r = view(routes, &sp);
    const DenseView h = view(H, "H", kValueTypes), y = view(Y, "Y", kValueTypes);
    if (y.rows != r.tokens) refuse("Y must have a row for each token");
    if (h.cols != y.cols || h.type != y.type) refuse("H and Y differ in columns or type");
    sp.add("H", h, false);
    sp.add("Y", y, true);
    add_weights(weights, "weights", r, h.type, false, &sp);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_combine(r, h, weights, y, (cudaStream_t)stream));
  });
}

int appt_combine_grad(const appt_routes* routes, const appt_dense* dY, const appt_dense* H,
                      const void* weights, const appt_dense* dH, void* dweights, int32_t device,
                      void* stream) {
  return guarded("appt_combine_grad", [&] {
    Spans sp;
    const RoutesView r = view(routes, &sp);
    const DenseView dy = view(dY, "dY", kValueTypes);
    if (dy.rows != r.tokens) refuse("dY must have a row for each token");
    if (r.tokens > 0 && !dH && !dweights) refuse("neither dH nor dweights is wanted");
    if (dweights && !H) refuse("dweights needs H");
    DenseView h, dh;
    if (dweights) {
      h = view(H, "H", kValueTypes);
      if (h.cols != dy.cols || h.type != dy.type) refuse("H and dY differ in columns or type");
      sp.add("H", h, false);
    }
    if (dH) {
      dh = view(dH, "dH", kValueTypes);
      if (dh.cols != dy.cols || dh.type != dy.type) refuse("dH and dY differ in columns or type");
      if (dweights && dh.rows != h.rows) refuse("dH and H differ in rows");
      sp.add("dH", dh, true);
    }
    sp.add("dY", dy, false);
    add_weights(weights, "weights", r, dy.type, false, &sp);
    add_weights(dweights, "dweights", r, dy.type, true, &sp);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_combine_grad(r, dy, dweights ? &h : nullptr, weights, dH ? &dh : nullptr,
                                 dweights, (cudaStream_t)stream));
  });
}

int appt_quantize(const appt_dense* X, int32_t gate, const int32_t* rows_ptr, const appt_scaled* Q,
                  int32_t device, void* stream) {
  return guarded("appt_quantize", [&] {
    Spans sp;
    const DenseView x = view(X, "X", kShortTypes);
    const ScaledView q = view(Q, "Q", true, 0, &sp);
    if (gate != APPT_GATE_NONE && gate != APPT_GATE_SILU) refuse("unknown gate");
    const int parts = gate == APPT_GATE_SILU ? 2 : 1;
    if (x.rows != q.q.rows || x.cols != parts * q.q.cols)
      refuse("X and Q differ in rows, or X has not the columns that the gate needs");
    if (rows_ptr && (uintptr_t)rows_ptr % 4) refuse("rows_ptr is not aligned to 4 bytes");
    sp.add("X", x, false);
    if (rows_ptr) sp.add("rows_ptr", rows_ptr, 1, 4, 4, false);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_quantize(x, parts == 2, rows_ptr, nullptr, q, (cudaStream_t)stream));
  });
}

int appt_dispatch_quantize(const appt_routes* routes, const appt_dense* X, const appt_scaled* Q,
                           int32_t device, void* stream) {
  return guarded("appt_dispatch_quantize", [&] {
    Spans sp;
    const RoutesView r = view(routes, &sp);
    const DenseView x = view(X, "X", kShortTypes);
    const ScaledView q = view(Q, "Q", true, 0, &sp);
    if (x.rows != r.tokens) refuse("X must have a row for each token");
    if (x.cols != q.q.cols) refuse("X and Q differ in columns");
    sp.add("X", x, false);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    note_launches(launch_quantize(x, false, nullptr, &r, q, (cudaStream_t)stream));
  });
}

int appt_scaled_product(const appt_scaled* A, const appt_blocks* W, const int32_t* group_ptr,
                        const appt_dense* Y, int32_t device, void* stream) {
  return guarded("appt_scaled_product", [&] {
    Spans sp;
    const ScaledView a = view(A, "A", false, 16, &sp);
    if (!W) refuse("W is null");
    BlocksView w;
    w.data = W->data;
    w.scale = W->scale;
    w.groups = W->groups;
    w.rows = W->rows;
    w.cols = W->cols;
    if (w.groups < 1 || w.groups > kMaxExperts)
      refuse("W: groups must lie in [1, " + std::to_string(kMaxExperts) + "]");
    if (w.rows < 1 || w.rows >= INT_MAX || w.cols < 1 || w.cols >= INT_MAX)
      refuse("W: rows and cols must lie in [1, 2^31 - 1)");
    w.ld = w.rows > 1 ? W->ld : (w.cols + 15) / 16 * 16;
    if (w.ld < w.cols || w.ld % 16 || w.ld >= (1ll << 38))
      refuse("W: ld must be a multiple of 16 and at least cols");
    if (w.rows > kLargest / w.ld) refuse("W: its rows reach further than any memory");
    w.group_stride = w.groups > 1 ? W->group_stride : (w.rows - 1) * w.ld + (w.cols + 15) / 16 * 16;
    if (w.group_stride < (w.rows - 1) * w.ld + w.cols || w.group_stride % 16 ||
        w.group_stride >= (1ll << 40))
      refuse("W: group_stride must be a multiple of 16 and at least one matrix");
    if (!w.data || (uintptr_t)w.data % 16 || !w.scale || (uintptr_t)w.scale % 4)
      refuse("W: data must be aligned to 16 bytes, scale to 4, neither null");
    if (a.q.cols != w.cols) refuse("A and W differ in columns");
    if (a.q.ld % 16) refuse("A: ld must be a multiple of 16");
    if (a.q.rows > 1 << 30 || w.rows > 1 << 30) refuse("more than 2^30 rows of A or W");
    const DenseView y = view(Y, "Y", kShortTypes);
    if (y.rows != a.q.rows || y.cols != w.rows) refuse("Y must be A's rows x W's rows");
    if (!group_ptr && w.groups != 1) refuse("group_ptr may be null with one group only");
    if (group_ptr && (uintptr_t)group_ptr % 4) refuse("group_ptr is not aligned to 4 bytes");
    const long long one = (w.rows - 1) * w.ld + w.cols;
    sp.add("W", w.data, w.groups, w.group_stride, one, false);
    const long long ns = 4 * w.groups * ((w.rows + kScaleBlock - 1) / kScaleBlock) *
                         ((w.cols + kScaleBlock - 1) / kScaleBlock);
    sp.add("W scale", w.scale, 1, ns, ns, false);
    sp.add("Y", y, true);
    if (group_ptr) sp.add("group_ptr", group_ptr, 1, 4 * (w.groups + 1), 4 * (w.groups + 1), false);
    check_overlap(sp);
    OnDevice on(device);
    check_resident(sp, device);
    if (y.rows == 0) return;
    note_launches(launch_scaled_product(a, w, group_ptr, y, on.sms, (cudaStream_t)stream));
  });
}

int appt_scaled_product_tile(int64_t rows, int64_t n, int64_t groups, int32_t sms,
                             int32_t* tile_rows, int32_t* tile_cols) {
  return guarded("appt_scaled_product_tile", [&] {
    if (rows < 0 || rows > 1 << 30 || n < 1 || n > 1 << 30 || groups < 1 || groups > kMaxExperts ||
        sms < 1 || sms > 1 << 16 || !tile_rows || !tile_cols)
      refuse("no product has these sizes, or a null output");
    const ProductTile t = scaled_product_tile(rows, n, groups, sms);
    *tile_rows = t.rows;
    *tile_cols = t.cols;
  });
}

void appt_scaled_product_give_up(int32_t on) { scaled_product_give_up(on != 0); }

int appt_scaled_product_status(int32_t device) {
  return guarded("appt_scaled_product_status", [&] {
    OnDevice on(device);
    check_cuda(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
    int gave_up = 0;
    check_cuda((cudaError_t)scaled_product_status(&gave_up), "reading the status");
    if (gave_up) refuse("a product gave up a wait", kErrDevice);
  });
}

}  // extern "C"
