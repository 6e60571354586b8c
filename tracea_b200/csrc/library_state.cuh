// Host state and helpers that the library's translation units share: the last error, the per-device state and its scratch,
// borrowed tensor views, the epilogue kinds and the environment knobs.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <mutex>
#include <string>
#include <thread>
#include <unordered_map>
#include <vector>

#include "../../include/tracea_b200.h"
#include "conv2d_sm100.cuh"

// Hidden: one copy for the library, none that another one could bind to.
namespace __attribute__((visibility("hidden"))) tb200_host {

// ------------------------------------------------------------------ last error (thread local)
inline thread_local std::string g_last_error;

inline void set_error(const char* fmt, ...) {
  char buf[1024];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
}

struct StatusError {
  TraceaStatus status;
};

#define TB_FAIL(status_, ...)        \
  do {                               \
    set_error(__VA_ARGS__);          \
    throw StatusError{status_};      \
  } while (0)

#define TB_CUDA(expr)                                                                   \
  do {                                                                                  \
    cudaError_t e_ = (expr);                                                            \
    if (e_ != cudaSuccess) {                                                            \
      TB_FAIL(TRACEA_CUDA_ERROR, "%s failed: %s", #expr, cudaGetErrorString(e_));       \
    }                                                                                   \
  } while (0)

// ------------------------------------------------------------------ driver entry points
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
typedef CUresult (*EncodeIm2colFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const int*, const int*,
                                   cuuint32_t, cuuint32_t, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

struct DeviceState {
  std::atomic<bool> ready{false};
  int dev = 0;
  int num_sms = 0;
  cudaMemPool_t pool = nullptr;
  uint32_t* status = nullptr;  // pinned, mapped: kernels write error codes the host reads directly
  std::mutex host_mu;          // one host-memory call at a time per device (it owns the copy streams below)
  // Scratch of the K-split schedule (fp32 partial sums, then the counters), one block per stream that has used it:
  // launches on one stream run one after another, so they can share a block, and the kernels leave the counters
  // at zero, so nothing has to be cleared between launches. Allocated once per stream with cudaMalloc.
  std::mutex ws_mu;
  std::unordered_map<unsigned long long, void*> split_ws;
  size_t split_partial_bytes = 0, split_counter_bytes = 0;
  // host-memory path only: copy streams and events for the chunked H2D / compute / D2H pipeline
  static constexpr int kMaxChunks = 16;
  cudaStream_t copy_in = nullptr, copy_out = nullptr;
  cudaEvent_t ev_entry = nullptr, ev_done = nullptr;
  cudaEvent_t ev_in[kMaxChunks] = {}, ev_out[kMaxChunks] = {};
};

constexpr int kMaxDevices = 64;
// Locking: each device's state is brought up once under its own mutex and is read-only afterwards, so host
// threads that drive different GPUs (or the same GPU on different streams) do not serialise on the call path:
// validation, tensor-map encoding and the launch itself run without any lock.
inline std::mutex g_dev_mu[kMaxDevices];
inline std::mutex g_driver_mu;
inline DeviceState g_dev[kMaxDevices];
// Test hooks (tracea_b200_test_hooks): a shortened wait limit and a producer that goes silent, so that a test can
// make a bounded wait run out without hanging anything. Off (0 / -1) unless a test sets them.
inline std::atomic<long long> g_test_wait_limit{0};
inline std::atomic<int> g_test_producer_stop{-1};
inline std::atomic<unsigned long long> g_kernel_launches{0};   // every kernel this library has launched (conv + layout adapters)
// the same, by kind: 0 general implicit-GEMM kernel, 1 its K-split instantiations, 2 resident-filter kernel, 3 layout adapters,
// 4 row-band kernel, 5 small-tile kernel; and 6, those of 0, 1 and 5 whose k-chunks run over whole filter rows; 7 conversions to
// and from the 4-bit format, 8 its matrix product, 9 the form of that for few rows, 10 norms
constexpr int kLaunchKinds = 11;
constexpr int kLaunchMxCopy = 7, kLaunchMxGemm = 8, kLaunchMxTokens = 9, kLaunchNorm = 10;
inline std::atomic<unsigned long long> g_launches_by_kind[kLaunchKinds];
inline EncodeTiledFn g_encode_tiled = nullptr;
inline EncodeIm2colFn g_encode_im2col = nullptr;

inline void load_driver_entry_points() {
  std::lock_guard<std::mutex> lock(g_driver_mu);
  if (g_encode_tiled != nullptr && g_encode_im2col != nullptr) return;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  TB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
  if (fn == nullptr || qres != cudaDriverEntryPointSuccess)
    TB_FAIL(TRACEA_CUDA_ERROR, "driver does not export cuTensorMapEncodeTiled");
  g_encode_tiled = reinterpret_cast<EncodeTiledFn>(fn);
  fn = nullptr;
  TB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeIm2col", &fn, cudaEnableDefault, &qres));
  if (fn == nullptr || qres != cudaDriverEntryPointSuccess)
    TB_FAIL(TRACEA_CUDA_ERROR, "driver does not export cuTensorMapEncodeIm2col");
  g_encode_im2col = reinterpret_cast<EncodeIm2colFn>(fn);
}

// The per-device state, brought up on first use (with `dev` current).
inline DeviceState& device_state(int dev) {
  if (dev < 0 || dev >= kMaxDevices) TB_FAIL(TRACEA_INVALID_PARAMS, "device_id %d out of range", dev);
  DeviceState& st = g_dev[dev];
  if (st.ready.load(std::memory_order_acquire)) return st;
  std::lock_guard<std::mutex> lock(g_dev_mu[dev]);
  if (st.ready.load(std::memory_order_relaxed)) return st;
  cudaDeviceProp prop;
  TB_CUDA(cudaGetDeviceProperties(&prop, dev));
  if (prop.major != 10)
    TB_FAIL(TRACEA_UNSUPPORTED_CONFIG,
            "device %d is sm_%d%d; this library only carries sm_100a kernels", dev, prop.major,
            prop.minor);
  st.dev = dev;
  st.num_sms = prop.multiProcessorCount;
  // the largest split any launch can ask for: 2 slots per worker of 256 x 256 fp32, 8 counter pairs per split tile
  st.split_partial_bytes = 2ull * st.num_sms * 256 * 256 * sizeof(float);
  st.split_counter_bytes = 2 * static_cast<size_t>(st.num_sms) * 8 * 2 * sizeof(uint32_t);   // up to two waves of tiles
  load_driver_entry_points();
  cudaMemPoolProps pp = {};
  pp.allocType = cudaMemAllocationTypePinned;
  pp.handleTypes = cudaMemHandleTypeNone;
  pp.location.type = cudaMemLocationTypeDevice;
  pp.location.id = dev;
  TB_CUDA(cudaMemPoolCreate(&st.pool, &pp));
  uint64_t keep = ~0ull;  // keep freed scratch cached in the pool instead of returning it to the OS
  TB_CUDA(cudaMemPoolSetAttribute(st.pool, cudaMemPoolAttrReleaseThreshold, &keep));
  TB_CUDA(cudaHostAlloc(reinterpret_cast<void**>(&st.status), 4 * sizeof(uint32_t),
                        cudaHostAllocMapped | cudaHostAllocPortable));
  memset(st.status, 0, 4 * sizeof(uint32_t));
  st.ready.store(true, std::memory_order_release);
  return st;
}

struct DeviceGuard {
  int prev = -1;
  bool switched = false;
  explicit DeviceGuard(int dev) {
    TB_CUDA(cudaGetDevice(&prev));
    if (prev != dev) {
      TB_CUDA(cudaSetDevice(dev));
      switched = true;
    }
  }
  ~DeviceGuard() {
    if (switched) cudaSetDevice(prev);
  }
};

// Stream-ordered scratch from the library's pool; released (stream-ordered) by the destructor.
struct Scratch {
  void* ptr = nullptr;
  cudaStream_t stream = nullptr;
  Scratch() = default;
  Scratch(const Scratch&) = delete;
  Scratch& operator=(const Scratch&) = delete;
  void alloc(DeviceState& st, size_t bytes, cudaStream_t s) {
    stream = s;
    TB_CUDA(cudaMallocFromPoolAsync(&ptr, bytes == 0 ? 16 : bytes, st.pool, s));
  }
  ~Scratch() {
    if (ptr != nullptr) cudaFreeAsync(ptr, stream);
  }
};

// The K-split scratch block of `stream` on this device (created on first use). A block's counters start at zero
// and every kernel leaves them at zero. Not for launches that are being captured into a graph: those take
// stream-ordered pool memory, which the graph owns.
inline void* split_workspace(DeviceState& st, cudaStream_t stream) {
  unsigned long long key = reinterpret_cast<unsigned long long>(stream);
  if (stream == cudaStreamPerThread)   // one handle, a different stream in every host thread
    key ^= static_cast<unsigned long long>(std::hash<std::thread::id>()(std::this_thread::get_id())) << 8;
  std::lock_guard<std::mutex> lock(st.ws_mu);
  auto it = st.split_ws.find(key);
  if (it != st.split_ws.end()) return it->second;
  void* base = nullptr;
  TB_CUDA(cudaMalloc(&base, st.split_partial_bytes + st.split_counter_bytes));
  TB_CUDA(cudaMemset(static_cast<char*>(base) + st.split_partial_bytes, 0, st.split_counter_bytes));
  st.split_ws.emplace(key, base);
  return base;
}

// After a kernel gave up a wait its counters may be anywhere: clear every block of the device.
inline void reset_split_workspaces(DeviceState& st) {
  std::lock_guard<std::mutex> lock(st.ws_mu);
  for (auto& kv : st.split_ws)
    cudaMemset(static_cast<char*>(kv.second) + st.split_partial_bytes, 0, st.split_counter_bytes);
}

// Reports, once, a kernel that gave up a bounded wait on this device since the last look (the words are in pinned host memory).
inline void fail_after_expired_wait(DeviceState& st) {
  if (st.status[0] != 0u) {
    const uint32_t code = st.status[0], blk = st.status[1], det = st.status[2];
    memset(st.status, 0, 4 * sizeof(uint32_t));
    cudaDeviceSynchronize();
    reset_split_workspaces(st);
    TB_FAIL(TRACEA_CUDA_ERROR,
            "an earlier kernel on device %d gave up a bounded wait (code %u, block %u, detail %u)",
            st.dev, code, blk, det);
  }
}

// ------------------------------------------------------------------ views
struct View4 {
  void* ptr = nullptr;
  long long shape[4] = {0, 0, 0, 0};
  long long stride[4] = {0, 0, 0, 0};
  TraceaDType dtype = TRACEA_DTYPE_FLOAT32;
  int device = -1;
};

inline int elem_size(TraceaDType t) {
  switch (t) {
    case TRACEA_DTYPE_FLOAT32: return 4;
    case TRACEA_DTYPE_FLOAT16: return 2;
    case TRACEA_DTYPE_BFLOAT16: return 2;
    default: return 0;
  }
}

inline const char* dtype_name(TraceaDType t) {
  switch (t) {
    case TRACEA_DTYPE_FLOAT32: return "float32";
    case TRACEA_DTYPE_FLOAT16: return "float16";
    case TRACEA_DTYPE_BFLOAT16: return "bfloat16";
    case TRACEA_DTYPE_INT32: return "int32";
    case TRACEA_DTYPE_INT8: return "int8";
    default: return "?";
  }
}

inline View4 load_view4(const TraceaTensorView& v, const char* name) {
  if (v.rank != 4) TB_FAIL(TRACEA_INVALID_PARAMS, "Expected 4D tensors (NCHW): %s has rank %u", name, v.rank);
  if (v.shape == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: shape array is NULL", name);
  View4 o;
  o.ptr = v.ptr;
  o.dtype = v.dtype;
  o.device = v.device_id;
  for (int i = 0; i < 4; ++i) {
    o.shape[i] = static_cast<long long>(v.shape[i]);
    // an empty batch (shape[0] == 0) is legal and is a no-op; every other extent must be positive
    if ((o.shape[i] <= 0 && !(i == 0 && o.shape[i] == 0)) || o.shape[i] > 0x7fffffffLL)
      TB_FAIL(TRACEA_INVALID_PARAMS, "%s: shape[%d] = %llu is out of range", name, i,
              (unsigned long long)v.shape[i]);
  }
  if (v.stride != nullptr) {
    for (int i = 0; i < 4; ++i) o.stride[i] = v.stride[i];
  } else {  // contiguous row-major, what tracea::TensorView builds (include/tracea.hpp:218-228)
    long long s = 1;
    for (int i = 3; i >= 0; --i) {
      o.stride[i] = s;
      s *= o.shape[i];
    }
  }
  for (int i = 0; i < 4; ++i)
    if (o.stride[i] < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: negative stride[%d]", name, i);
  return o;
}

// Number of elements from the first to the last addressed element, inclusive.
inline long long span_elems(const View4& v) {
  long long s = 1;
  for (int i = 0; i < 4; ++i) s += (v.shape[i] - 1) * v.stride[i];
  return s;
}
inline long long num_elems(const View4& v) { return v.shape[0] * v.shape[1] * v.shape[2] * v.shape[3]; }

// Strides of extent-1 dimensions carry no information (torch reports arbitrary values for them);
// when the channel axis is innermost, rewrite them to the dense channels-last values so that the
// layout tests below and the TMA stride rules see a consistent picture.
inline void canon_channels_last(View4& v) {
  if (v.shape[1] != 1 && v.stride[1] != 1) return;
  if (v.shape[1] == 1) v.stride[1] = 1;
  if (v.shape[3] == 1) v.stride[3] = v.shape[1];
  if (v.shape[2] == 1) v.stride[2] = v.shape[3] * v.stride[3];
  if (v.shape[0] == 1) v.stride[0] = v.shape[2] * v.stride[2];
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ------------------------------------------------------------------ epilogue decoding
struct Epilogue {
  bool bias = false;
  bool residual = false;
  int act = tb200::kActNone;
};

// Kind -> op list, after src/interface/c_bindings.rs:144-197.
inline Epilogue decode_epilogue(TraceaEpilogueKind kind, bool have_bias, bool have_res) {
  Epilogue e;
  switch (kind) {
    case TRACEA_EPILOGUE_IDENTITY: break;
    case TRACEA_EPILOGUE_BIAS_ADD: e.bias = have_bias; break;
    case TRACEA_EPILOGUE_RELU: e.act = tb200::kActRelu; break;
    case TRACEA_EPILOGUE_GELU: e.act = tb200::kActGelu; break;
    case TRACEA_EPILOGUE_SILU: e.act = tb200::kActSilu; break;
    case TRACEA_EPILOGUE_BIAS_RELU: e.bias = have_bias; e.act = tb200::kActRelu; break;
    case TRACEA_EPILOGUE_BIAS_SILU:
      // the reference emits the fused BiasAddSiLU functor only when a bias is present
      e.bias = have_bias;
      e.act = have_bias ? tb200::kActSilu : tb200::kActNone;
      break;
    case TRACEA_EPILOGUE_RESIDUAL: e.residual = have_res; break;
    case TRACEA_EPILOGUE_RESIDUAL_RELU: e.residual = have_res; e.act = tb200::kActRelu; break;
    case TRACEA_EPILOGUE_BIAS_RESIDUAL_RELU:
      e.bias = have_bias; e.residual = have_res; e.act = tb200::kActRelu; break;
    case TRACEA_EPILOGUE_BIAS_RESIDUAL: e.bias = have_bias; e.residual = have_res; break;
    default:
      TB_FAIL(TRACEA_INVALID_PARAMS, "unknown epilogue kind %d", static_cast<int>(kind));
  }
  return e;
}

// ------------------------------------------------------------------ environment knobs
inline int env_int(const char* name, int dflt) {
  const char* v = getenv(name);
  return (v != nullptr && *v != '\0') ? atoi(v) : dflt;
}

// Bring-up / test knobs, read from the environment once per process (a getenv per knob per call is a measurable
// part of the ~6 us a call costs on the host). TRACEA_B200_HOST_CHUNKS is read per call and is not in here.
struct Knobs {
  int force_bn, force_stages, force_chunk, no_tma_store, no_tma_residual, tiled_a, force_staging, no_window,
      pair, rows2, panel, pdl, split_k, no_window3, no_row_band;
};
inline const Knobs& knobs() {
  static const Knobs k = {
      env_int("TRACEA_B200_FORCE_BN", 0),      env_int("TRACEA_B200_FORCE_STAGES", 0),
      env_int("TRACEA_B200_FORCE_CHUNK", 0),   env_int("TRACEA_B200_NO_TMA_STORE", 0),
      env_int("TRACEA_B200_NO_TMA_RESIDUAL", 0), env_int("TRACEA_B200_TILED_A", 0),
      env_int("TRACEA_B200_FORCE_STAGING", 0), env_int("TRACEA_B200_NO_WINDOW", 0),
      env_int("TRACEA_B200_PAIR", -1),         env_int("TRACEA_B200_ROWS2", -1),
      env_int("TRACEA_B200_PANEL", 0),         env_int("TRACEA_B200_PDL", 1),
      env_int("TRACEA_B200_SPLIT_K", 0),       env_int("TRACEA_B200_NO_RESIDENT_FILTER", 0),
      env_int("TRACEA_B200_NO_ROW_BAND", 0)};
  return k;
}

// ------------------------------------------------------------------ matrices
struct Rank2 {
  long long shape[2];
  long long stride[2];
};

inline Rank2 load_rank2(const TraceaTensorView& v, const char* name) {
  if (v.rank != 2) TB_FAIL(TRACEA_INVALID_PARAMS, "Expected 2D tensors: %s has rank %u", name, v.rank);
  if (v.shape == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: shape array is NULL", name);
  Rank2 r;
  for (int i = 0; i < 2; ++i) {
    r.shape[i] = static_cast<long long>(v.shape[i]);
    if (r.shape[i] < 0 || r.shape[i] > 0x7fffffffLL)
      TB_FAIL(TRACEA_INVALID_PARAMS, "%s: shape[%d] = %llu is out of range", name, i, (unsigned long long)v.shape[i]);
  }
  r.stride[0] = v.stride != nullptr ? v.stride[0] : r.shape[1];
  r.stride[1] = v.stride != nullptr ? v.stride[1] : 1;
  if (r.stride[0] < 0 || r.stride[1] < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: negative stride", name);
  return r;
}

// ------------------------------------------------------------------ the C boundary
template <typename F>
TraceaStatus guarded(const char* what, F&& f) {
  // mirrors the catch_unwind wrapper of tracea-ffi/src/lib.rs:130-141: nothing escapes the C boundary
  try {
    f();
    return TRACEA_SUCCESS;
  } catch (const StatusError& e) {
    return e.status;
  } catch (const std::exception& e) {
    set_error("Exception in %s: %s", what, e.what());
    return TRACEA_UNKNOWN_ERROR;
  } catch (...) {
    set_error("Unknown exception in %s", what);
    return TRACEA_UNKNOWN_ERROR;
  }
}

}  // namespace tb200_host
