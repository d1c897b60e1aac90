// Host-side pieces shared by the library's translation units: status exceptions and their
// conversion at the C boundary, the context, kernel launches, device allocations and the
// driver's tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdlib>
#include <exception>
#include <map>
#include <mutex>
#include <new>
#include <string>
#include <thread>
#include <utility>
#include <vector>

#include "../../include/woodcock_b200.h"

// ============================================================================ errors

namespace {

struct WcError {
  wc_status st;
  std::string msg;
};

[[noreturn]] void fail(wc_status st, const std::string& msg) { throw WcError{st, msg}; }

#define CUDA_TRY(x)                                                                                  \
  do {                                                                                               \
    cudaError_t e_ = (x);                                                                            \
    if (e_ != cudaSuccess) fail(e_ == cudaErrorMemoryAllocation ? WC_ERR_OOM : WC_ERR_CUDA,          \
                                std::string(#x) + ": " + cudaGetErrorString(e_));                    \
  } while (0)

}  // namespace

// The last failure's message, by thread: paged calls of several threads share a context. A thread that
// had no failure of its own is told the latest of any.
class LastError {
 public:
  void set(const char* msg) noexcept {
    try {
      std::lock_guard<std::mutex> lock(mu_);
      latest_ = msg;
      of_[std::this_thread::get_id()] = latest_;
    } catch (...) {  // no memory for the words: the status still stands
    }
  }
  const char* get() const noexcept {  // valid until the calling thread's next failure
    try {
      std::lock_guard<std::mutex> lock(mu_);
      return of_.emplace(std::this_thread::get_id(), latest_).first->second.c_str();
    } catch (...) {
      return "host allocation failed";
    }
  }

 private:
  mutable std::mutex mu_;
  mutable std::map<std::thread::id, std::string> of_;
  std::string latest_;
};

// ============================================================================ context

struct RopeTable {
  float2* ptr = nullptr;
  int max_pos = 0;
};

// CUDA-event marks around kernels of a profiled round (a separate graph from the timed one).
enum ProfKind { PK_QKV, PK_ATTN, PK_O, PK_GU, PK_DOWN, PK_HEAD, PK_DRAFT_HEAD, PK_DRAFT_LAYER, PK_COUNT };
constexpr int PK_SLOTS = 16;  // entries of the profile arrays in the C ABI

struct Profiler {
  std::vector<cudaEvent_t> pool;
  size_t next = 0;
  std::vector<std::pair<int, std::pair<cudaEvent_t, cudaEvent_t>>> marks;
  cudaEvent_t open[PK_COUNT] = {};
  cudaEvent_t take() {
    if (next == pool.size()) {
      cudaEvent_t e;
      cudaEventCreate(&e);
      pool.push_back(e);
    }
    return pool[next++];
  }
  ~Profiler() {
    for (auto e : pool) cudaEventDestroy(e);
  }
};

struct wc_ctx {
  int device = 0;
  cudaStream_t stream = nullptr;
  bool own_stream = false;
  int num_sms = 148;
  LastError err;
  int* d_err = nullptr;  // device error word of the ops API
  std::atomic<uint64_t> launches{0};
  std::atomic<bool> capturing{false};  // on `stream`
  std::atomic<uint64_t> capture_launches{0};
  std::map<std::pair<int, uint32_t>, RopeTable> rope;
  double* pw = nullptr;
  double* qw = nullptr;
  int pw_n = 0;
  int occ_gemv[3] = {1, 1, 1};  // [0] fp32, [1] bf16 NT=1, [2] bf16 NT=2
  size_t max_smem = 0;
  Profiler* prof = nullptr;  // set while a profiled round is being captured
  bool pdl = true;           // programmatic dependent launch between round kernels
  int attn_mode = 4;         // bf16 caches: 4 the cluster kernel (attention_dec.cuh), 2 the
                             // split-sequence kernel (attention_split.cuh; always used for drafted
                             // tree levels), 1 split-KV mma kernel, 0 CUDA cores
  float* as_part_o = nullptr;   // attention_split partial states: [16 KV heads][AS_MAXS + 1][AS_MAXR][128]
  float* as_part_ml = nullptr;  //   and their (m, l): [16][AS_MAXS + 1][AS_MAXR][2]
  int* as_counters = nullptr;   //   per-KV-head arrivals (zero between launches)
  int attn_split_pos = 256;     // capacity positions per prefix block (WC_ATTN_SPLIT_POS)
  int gemv_blocks_per_sm = 1;
  bool gemv_wide = true;                 // 80 KB activation chunks for K up to 2560 (WC_GEMV_WIDE=0: split K)
  bool gemv_acs = true;                  // whole-K blocks with streamed activation pieces (WC_GEMV_ACS=0: split K)
  bool gemv_prefetch = false;            // L2 prefetch of the next GEMV's weights (WC_GEMV_PREFETCH=1;
                                         // measured 1.6% slower on the C3 round: it competes with the
                                         // dependent loads of the kernels in between)
  size_t gemv_prefetch_cap = 64u << 20;  // bytes prefetched at most
  float* gv_partial = nullptr;           // split-K partial sums
  size_t gv_partial_n = 0;               // floats
  int* gv_counters = nullptr;            // split-K arrival counters (zero between launches)
  int gv_counters_n = 0;
  void* pw_scratch = nullptr;            // wc_probs_from_logits: parameters + row thresholds
  int pw_rows = 0;
  uint32_t* lin_xf = nullptr;  // input fragments of the ops-API linear
  int lin_xf_k = 0;
  bool lin_xf_bf16 = false;
};

namespace {

template <class F>
wc_status guard(wc_ctx* ctx, F&& f) {
  try {
    f();
    return WC_OK;
  } catch (const WcError& e) {
    if (ctx) ctx->err.set(e.msg.c_str());
    return e.st;
  } catch (const std::bad_alloc&) {
    if (ctx) ctx->err.set("host allocation failed");
    return WC_ERR_OOM;
  } catch (const std::exception& e) {
    if (ctx) ctx->err.set(e.what());
    return WC_ERR_IO;
  }
}

void prof_begin(wc_ctx* ctx, int kind) {
  if (!ctx->prof) return;
  cudaEvent_t e = ctx->prof->take();
  // external event nodes: a plain record inside stream capture is only a dependency marker
  if (ctx->capturing) cudaEventRecordWithFlags(e, ctx->stream, cudaEventRecordExternal);
  else cudaEventRecord(e, ctx->stream);
  ctx->prof->open[kind] = e;
}

void prof_end(wc_ctx* ctx, int kind) {
  if (!ctx->prof || !ctx->prof->open[kind]) return;
  cudaEvent_t e = ctx->prof->take();
  if (ctx->capturing) cudaEventRecordWithFlags(e, ctx->stream, cudaEventRecordExternal);
  else cudaEventRecord(e, ctx->stream);
  ctx->prof->marks.push_back({kind, {ctx->prof->open[kind], e}});
  ctx->prof->open[kind] = nullptr;
}

void count_launch(wc_ctx* ctx, cudaStream_t stream) {
  if (ctx->capturing && stream == ctx->stream) ++ctx->capture_launches;
  else ++ctx->launches;
}

void check_launch(wc_ctx* ctx, const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) fail(WC_ERR_CUDA, std::string("launch of ") + what + " failed: " + cudaGetErrorString(e));
  count_launch(ctx, ctx->stream);
}

// Launch with optional programmatic dependent launch (the kernel must pdl_wait() before it
// reads anything the previous kernel writes) and an optional cluster along x.
template <typename... KArgs, typename... Args>
void launch_on(wc_ctx* ctx, cudaStream_t stream, const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block,
               size_t smem, bool pdl, int cluster_x, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (pdl && ctx->pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  if (cluster_x > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = cluster_x;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  if (e != cudaSuccess) fail(WC_ERR_CUDA, std::string("launch of ") + what + ": " + cudaGetErrorString(e));
  count_launch(ctx, stream);
}

// The same on the context's stream.
template <typename... KArgs, typename... Args>
void launch_ex(wc_ctx* ctx, const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, bool pdl,
               int cluster_x, Args&&... args) {
  launch_on(ctx, ctx->stream, what, kernel, grid, block, smem, pdl, cluster_x, std::forward<Args>(args)...);
}

void* dalloc(size_t bytes) {
  if (bytes == 0) bytes = 16;
  void* p = nullptr;
  const cudaError_t e = cudaMalloc(&p, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    fail(WC_ERR_OOM, "cudaMalloc(" + std::to_string(bytes) + ") failed: " + cudaGetErrorString(e));
  }
  return p;
}

void dfree(void* p) {
  if (p) cudaFree(p);
}

// A call's device where it is not the current one; the current one comes back at its end.
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(int device) {
    int cur = 0;
    CUDA_TRY(cudaGetDevice(&cur));
    if (cur != device) {
      CUDA_TRY(cudaSetDevice(device));
      before = cur;
    }
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || !p || q != cudaDriverEntryPointSuccess)
      fail(WC_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

}  // namespace
