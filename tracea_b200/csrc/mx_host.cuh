// Host helpers of the 4-bit microscaled operators and the norms: their views, their checks and the launch.
#pragma once
#include "library_state.cuh"
#include "mx_format.cuh"

namespace __attribute__((visibility("hidden"))) tb200_host {

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// ------------------------------------------------------------------ views
struct Matrix {
  char* ptr;
  long long rows, cols, row_stride, col_stride;   // strides in elements
  TraceaDType dtype;
  int es;
};

inline Matrix load_matrix(const TraceaTensorView& v, const char* name, int dev) {
  const Rank2 r = load_rank2(v, name);
  Matrix m;
  m.ptr = static_cast<char*>(v.ptr);
  m.rows = r.shape[0];
  m.cols = r.shape[1];
  m.row_stride = r.stride[0];
  m.col_stride = r.shape[1] == 1 ? 1 : r.stride[1];
  if (m.rows == 1) m.row_stride = m.cols;           // an extent of 1 has no stride
  m.dtype = v.dtype;
  m.es = elem_size(v.dtype);
  if (m.es == 0) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: unsupported dtype %s", name, dtype_name(v.dtype));
  if (v.device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is on device %d, expected %d", name, v.device_id, dev);
  if (m.rows > 0 && m.cols > 0 && v.ptr == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s has a NULL pointer", name);
  if ((reinterpret_cast<uintptr_t>(v.ptr) & (m.es - 1)) != 0)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s is not aligned to its elements", name);
  return m;
}

inline void check_output(const Matrix& m, const char* name) {
  if ((m.rows > 1 && m.cols > 0 && m.row_stride == 0) || (m.cols > 1 && m.rows > 0 && m.col_stride == 0) ||
      (m.rows > 1 && m.col_stride == 1 && m.row_stride < m.cols))
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s: its rows overlap", name);
}

// Whether eight columns at a time can be moved in 16-byte accesses.
inline bool rows_of_8(const Matrix& m) {
  return m.col_stride == 1 && aligned16(m.ptr) && m.row_stride * m.es % 16 == 0;
}
// Bytes a lane may move at once along rows: 16, 8, 4, or one element.
inline int row_vec(const void* ptr, long long row_stride, long long cols, int es) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
  if (a % 16 == 0 && row_stride * es % 16 == 0 && cols * es % 16 == 0) return 16;
  if (a % 8 == 0 && row_stride * es % 8 == 0 && cols * es % 8 == 0) return 8;
  if (a % 4 == 0 && row_stride * es % 4 == 0 && cols * es % 4 == 0) return 4;
  return es;
}

// Row numbers, and those of rows a CTA looks ahead to, are 32-bit.
inline void check_rows(const Matrix& m, const char* name) {
  if (m.rows > 0x7fffff00LL) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld rows, at most %lld", name, m.rows, 0x7fffff00LL);
}

struct Mx {
  uint8_t *data, *scales;
  long long rows, cols, blocks, k_tiles;
};

inline Mx load_mx(const TraceaMxMatrix& v, const char* name, int dev) {
  Mx m;
  m.data = static_cast<uint8_t*>(v.data);
  m.scales = static_cast<uint8_t*>(v.scales);
  if (v.rows > 0x7fffff00ULL || v.cols == 0 || v.cols > 0x7fffff00ULL)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s: %llu x %llu is out of range", name, (unsigned long long)v.rows, (unsigned long long)v.cols);
  m.rows = static_cast<long long>(v.rows);
  m.cols = static_cast<long long>(v.cols);
  m.blocks = ceil_div(m.cols, tb200::kMxBlock);
  m.k_tiles = ceil_div(m.cols, tb200::kMxTileCols);
  if (v.device_id != dev || dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is on device %d, expected %d", name, v.device_id, dev);
  if (m.rows > 0 && (m.data == nullptr || m.scales == nullptr)) TB_FAIL(TRACEA_INVALID_PARAMS, "%s has a NULL pointer", name);
  if (!aligned16(m.data) || !aligned16(m.scales)) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: data and scales must be 16-byte aligned", name);
  return m;
}

inline void check_mx_shape(const Mx& m, const char* name, long long rows, long long cols) {
  if (m.rows != rows || m.cols != cols)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s is [%lld,%lld], expected [%lld,%lld]", name, m.rows, m.cols, rows, cols);
}

inline unsigned grid_of(long long blocks) {
  if (blocks > 0x7fffffffLL) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "tensor too large");
  return static_cast<unsigned>(blocks);
}

// Every kernel here is a programmatic launch: it may come up beside the one in front of it, and waits for that before it touches
// global memory.
template <typename Kernel, typename... Args>
void launch(Kernel kern, dim3 grid, int threads, int smem, int cluster, int kind, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (knobs().pdl != 0) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  TB_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  TB_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  g_launches_by_kind[kind].fetch_add(1, std::memory_order_relaxed);
}

template <typename F>
void by_dtype(TraceaDType t, F&& f) {
  switch (t) {
    case TRACEA_DTYPE_BFLOAT16: f(__nv_bfloat16{}); break;
    case TRACEA_DTYPE_FLOAT16: f(__half{}); break;
    default: f(0.0f); break;
  }
}

}  // namespace tb200_host
