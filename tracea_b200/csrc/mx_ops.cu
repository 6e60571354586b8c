// Host side of the 4-bit microscaled operators and of the norms around a block: tracea_mx_quantize, tracea_mx_dequantize,
// tracea_mx_gemm, tracea_mx_linear, tracea_block_norm, tracea_block_norm_add. The reference has no counterpart of any of them.
#include "library_state.cuh"
#include "block_norm_sm100.cuh"
#include "mx_format.cuh"
#include "mx_gemm_sm100.cuh"

namespace {

using namespace tb200_host;

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// ------------------------------------------------------------------ views
struct Matrix {
  char* ptr;
  long long rows, cols, row_stride, col_stride;   // strides in elements
  TraceaDType dtype;
  int es;
};

Matrix load_matrix(const TraceaTensorView& v, const char* name, int dev) {
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

void check_output(const Matrix& m, const char* name) {
  if ((m.rows > 1 && m.cols > 0 && m.row_stride == 0) || (m.cols > 1 && m.rows > 0 && m.col_stride == 0) ||
      (m.rows > 1 && m.col_stride == 1 && m.row_stride < m.cols))
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s: its rows overlap", name);
}

// Whether eight columns at a time can be moved in 16-byte accesses.
bool rows_of_8(const Matrix& m) {
  return m.col_stride == 1 && aligned16(m.ptr) && m.row_stride * m.es % 16 == 0;
}
// Bytes a lane may move at once along rows: 16, 4, or one element.
int row_vec(const void* ptr, long long row_stride, long long cols, int es) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
  if (a % 16 == 0 && row_stride * es % 16 == 0 && cols * es % 16 == 0) return 16;
  if (a % 4 == 0 && row_stride * es % 4 == 0 && cols * es % 4 == 0) return 4;
  return es;
}

struct Mx {
  uint8_t *data, *scales;
  long long rows, cols, blocks, k_tiles;
};

Mx load_mx(const TraceaMxMatrix& v, const char* name, int dev) {
  Mx m;
  m.data = static_cast<uint8_t*>(v.data);
  m.scales = static_cast<uint8_t*>(v.scales);
  if (v.rows > 0x7fffffffULL || v.cols == 0 || v.cols > 0x7fffff00ULL)
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

void check_mx_shape(const Mx& m, const char* name, long long rows, long long cols) {
  if (m.rows != rows || m.cols != cols)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s is [%lld,%lld], expected [%lld,%lld]", name, m.rows, m.cols, rows, cols);
}

unsigned grid_of(long long blocks) {
  if (blocks > 0x7fffffffLL) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "tensor too large");
  return static_cast<unsigned>(blocks);
}

// Every kernel here is a programmatic launch: it may come up beside the one in front of it, and waits for that before it touches
// global memory.
template <typename Kernel, typename... Args>
void launch(Kernel kern, unsigned grid, int threads, int smem, int cluster, int kind, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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

// ------------------------------------------------------------------ matrix <-> format
tb200::MxCopyArgs copy_args(const Matrix& m, const Mx& q) {
  tb200::MxCopyArgs a;
  memset(&a, 0, sizeof(a));
  a.scales = q.scales;
  a.row_stride = m.row_stride;
  a.col_stride = m.col_stride;
  a.M = m.rows;
  a.K = static_cast<int>(m.cols);
  a.blocks = static_cast<int>(q.blocks);
  a.k_tiles = static_cast<int>(q.k_tiles);
  a.chunks = static_cast<int>(ceil_div(m.cols, 256));
  return a;
}
unsigned copy_grid(const tb200::MxCopyArgs& a) {
  return grid_of(ceil_div(ceil_div(a.M, tb200::kMxTileRows) * 32 * a.chunks, tb200::kMxCopyThreads / 32));
}

void quantize(const Matrix& x, const Mx& q, cudaStream_t stream) {
  tb200::MxCopyArgs a = copy_args(x, q);
  a.src = x.ptr;
  a.dst = q.data;
  by_dtype(x.dtype, [&](auto tag) {
    using T = decltype(tag);
    launch(rows_of_8(x) && x.cols % 8 == 0 ? tb200::mx_quantize_kernel<T, true> : tb200::mx_quantize_kernel<T, false>, copy_grid(a),
           tb200::kMxCopyThreads, 0, 1, kLaunchMxCopy, stream, a);
  });
}

void mx_quantize_checked(const TraceaTensorView& xv, const TraceaMxMatrix* qv, void* stream) {
  if (qv == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "Null pointer in quantize arguments");
  const int dev = xv.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "tracea_mx_quantize takes device tensors (device_id >= 0)");
  const Matrix x = load_matrix(xv, "x", dev);
  const Mx q = load_mx(*qv, "q", dev);
  check_mx_shape(q, "q", x.rows, x.cols);
  if (x.rows == 0) return;
  DeviceGuard guard(dev);
  device_state(dev);
  quantize(x, q, static_cast<cudaStream_t>(stream));
}

void mx_dequantize_checked(const TraceaMxMatrix& qv, const TraceaTensorView* outv, void* stream) {
  if (outv == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "Null pointer in dequantize arguments");
  const int dev = qv.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "tracea_mx_dequantize takes device tensors (device_id >= 0)");
  const Mx q = load_mx(qv, "q", dev);
  const Matrix out = load_matrix(*outv, "out", dev);
  check_mx_shape(q, "q", out.rows, out.cols);
  check_output(out, "out");
  if (out.rows == 0) return;
  DeviceGuard guard(dev);
  device_state(dev);
  tb200::MxCopyArgs a = copy_args(out, q);
  a.src = q.data;
  a.dst = out.ptr;
  by_dtype(out.dtype, [&](auto tag) {
    using T = decltype(tag);
    launch(rows_of_8(out) && out.cols % 8 == 0 ? tb200::mx_dequantize_kernel<T, true> : tb200::mx_dequantize_kernel<T, false>,
           copy_grid(a), tb200::kMxCopyThreads, 0, 1, kLaunchMxCopy, static_cast<cudaStream_t>(stream), a);
  });
}

// ------------------------------------------------------------------ product
void encode(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion, const char* what) {
  const cuuint32_t ones[3] = {1u, 1u, 1u};
  const CUresult r = g_encode_tiled(m, type, static_cast<cuuint32_t>(rank), const_cast<void*>(ptr), dims, strides, box, ones,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) TB_FAIL(TRACEA_CUDA_ERROR, "cuTensorMapEncodeTiled (%s) failed with %d", what, (int)r);
}
// 128 bytes of `box_rows` rows of codes
void encode_codes(CUtensorMap* m, const Mx& q, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(16 * q.blocks), static_cast<cuuint64_t>(q.rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(16 * q.blocks)};
  const cuuint32_t box[2] = {128u, static_cast<cuuint32_t>(box_rows)};
  encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, q.data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, "codes");
}
// two tiles along K of `row_tiles` tiles of scales
void encode_scales(CUtensorMap* m, const Mx& q, int row_tiles) {
  const cuuint64_t dims[3] = {tb200::kMxTileBytes / 4, static_cast<cuuint64_t>(q.k_tiles),
                              static_cast<cuuint64_t>(ceil_div(q.rows, tb200::kMxTileRows))};
  const cuuint64_t strides[2] = {tb200::kMxTileBytes, static_cast<cuuint64_t>(q.k_tiles * tb200::kMxTileBytes)};
  const cuuint32_t box[3] = {tb200::kMxTileBytes / 4, 2u, static_cast<cuuint32_t>(row_tiles)};
  encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, q.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, "scales");
}

struct Product {
  Mx a, w;
  Epilogue epi;
  const void* bias = nullptr;
  bool bias_is_f32 = false;
  Matrix out{}, residual{};
  Mx out_mx{};
  bool to_mx = false;
};

std::atomic<bool> g_mx_attr_set[kMaxDevices][3][3][3];

template <typename OutT, int BN, bool kPair, int kStore>
void launch_mx_gemm(DeviceState& st, int dt, const Product& p, cudaStream_t stream) {
  constexpr int kBnIdx = BN / 64 - 1;
  auto kern = tb200::mx_gemm_sm100_kernel<OutT, BN, kPair, kStore>;
  std::atomic<bool>& attr_done = g_mx_attr_set[st.dev][dt][kBnIdx][kStore];
  if (!attr_done.load(std::memory_order_relaxed)) {
    TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
    attr_done.store(true, std::memory_order_relaxed);
  }
  const long long M = p.a.rows, N = p.w.rows, K = p.a.cols;
  constexpr int kTileM = kPair ? 256 : 128;
  tb200::MxGemmArgs g;
  memset(&g, 0, sizeof(g));
  g.M = static_cast<int>(M);
  g.N = static_cast<int>(N);
  g.k_iters = static_cast<int>(ceil_div(K, 256));
  const long long m_tiles = ceil_div(M, kTileM), n_tiles = ceil_div(N, BN);
  const long long panel = std::min<long long>(n_tiles, 8);
  if (m_tiles * n_tiles > 0x3fffffffLL) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "too many tiles");
  g.num_m_tiles = static_cast<int>(m_tiles);
  g.num_n_tiles = static_cast<int>(n_tiles);
  g.panel_width = static_cast<int>(panel);
  g.panel_tiles = static_cast<int>(m_tiles * panel);
  constexpr int kDepth = kStore == tb200::kMxStoreTma ? 2 : (kStore == tb200::kMxStoreRows ? 1 : 0);
  const int room = 232448 - tb200::mx_smem_bytes(BN, 0, kPair, kDepth);
  int stages = std::min(room / tb200::mx_stage_bytes(BN, kPair), tb200::kMxMaxStages);
  stages = std::min(stages, (512 - 2 * BN) / tb200::mx_scale_cols(BN));
  g.num_stages = stages;
  g.idesc = tb200::ptx::make_mx_idesc(kTileM, BN);
  g.bias = p.bias;
  g.bias_is_f32 = p.bias_is_f32 ? 1 : 0;
  g.act = p.epi.act;
  g.status = st.status;
  const long long limit = g_test_wait_limit.load(std::memory_order_relaxed);
  g.wait_limit = limit > 0 ? limit : tb200::kWaitLimitCycles;
  g.test_producer_stop = g_test_producer_stop.load(std::memory_order_relaxed);
  CUtensorMap ta, tw, tsa, tsw, to;
  encode_codes(&ta, p.a, 128);
  encode_codes(&tw, p.w, kPair ? BN / 2 : BN);
  encode_scales(&tsa, p.a, 1);
  encode_scales(&tsw, p.w, tb200::mx_b_scale_tiles(BN));
  memset(&to, 0, sizeof(to));
  if constexpr (kStore == tb200::kMxStoreMx) {
    g.out = p.out_mx.data;
    g.out_scales = p.out_mx.scales;
    g.out_blocks = static_cast<int>(p.out_mx.blocks);
    g.out_k_tiles = static_cast<int>(p.out_mx.k_tiles);
  } else {
    g.out = p.out.ptr;
    g.out_stride = p.out.row_stride;
    g.out_vec = row_vec(p.out.ptr, p.out.row_stride, N, sizeof(OutT));
    if (p.epi.residual) {
      g.residual = p.residual.ptr;
      g.res_stride = p.residual.row_stride;
      g.res_vec = row_vec(p.residual.ptr, p.residual.row_stride, N, sizeof(OutT));
    }
    if constexpr (kStore == tb200::kMxStoreTma) {
      const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
      const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.out.row_stride) * sizeof(OutT)};
      const cuuint32_t box[2] = {128u / sizeof(OutT), 32u};
      const CUtensorMapDataType type = dt == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : (dt == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32);
      encode(&to, type, 2, p.out.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, "output");
    }
  }
  const long long workers = std::min<long long>(m_tiles * n_tiles, kPair ? st.num_sms / 2 : st.num_sms);
  launch(kern, grid_of(kPair ? 2 * workers : workers), tb200::mx_threads(kPair), tb200::mx_smem_bytes(BN, stages, kPair, kDepth),
         kPair ? 2 : 1, kLaunchMxGemm, stream, ta, tw, tsa, tsw, to, g);
}

void mx_product(DeviceState& st, const Product& p, cudaStream_t stream) {
  const int force = env_int("TRACEA_B200_MX_BN", 0);
  const long long M = p.a.rows, N = p.w.rows;
  const int bn = force != 0 ? force : (M > 128 && ceil_div(M, 256) * ceil_div(N, 192) >= st.num_sms / 2 ? 192 : (N > 64 ? 128 : 64));
  auto tiled = [&](auto tag, int dt, auto store) {
    using T = decltype(tag);
    constexpr int kStore = decltype(store)::value;
    if (bn == 192) launch_mx_gemm<T, 192, true, kStore>(st, dt, p, stream);
    else if (bn == 128) launch_mx_gemm<T, 128, false, kStore>(st, dt, p, stream);
    else launch_mx_gemm<T, 64, false, kStore>(st, dt, p, stream);
  };
  if (p.to_mx) {
    tiled(__nv_bfloat16{}, 0, std::integral_constant<int, tb200::kMxStoreMx>{});
    return;
  }
  const bool tma = aligned16(p.out.ptr) && p.out.row_stride * p.out.es % 16 == 0;
  by_dtype(p.out.dtype, [&](auto tag) {
    const int dt = p.out.dtype == TRACEA_DTYPE_BFLOAT16 ? 0 : (p.out.dtype == TRACEA_DTYPE_FLOAT16 ? 1 : 2);
    if (tma) tiled(tag, dt, std::integral_constant<int, tb200::kMxStoreTma>{});
    else tiled(tag, dt, std::integral_constant<int, tb200::kMxStoreRows>{});
  });
}

// The arguments that tracea_mx_gemm and tracea_mx_linear share; M x K is the input's shape.
Product check_product(int dev, long long M, long long K, const TraceaMxMatrix& wv, const TraceaTensorView* biasv,
                      const TraceaTensorView* resv, const TraceaTensorView* cv, const TraceaMxMatrix* cq,
                      const TraceaGemmParams& gp) {
  if ((cv == nullptr) == (cq == nullptr)) TB_FAIL(TRACEA_INVALID_PARAMS, "exactly one of c and c_mx must be given");
  Product p;
  p.w = load_mx(wv, "w", dev);
  if (p.w.cols != K) TB_FAIL(TRACEA_INVALID_PARAMS, "Inner dimension mismatch: a is [%lld,%lld], w is [%lld,%lld]", M, K, p.w.rows, p.w.cols);
  const long long N = p.w.rows;
  if (N == 0) TB_FAIL(TRACEA_INVALID_PARAMS, "w has no rows");
  p.epi = decode_epilogue(gp.epilogue, biasv != nullptr, resv != nullptr);
  TraceaDType dtype = TRACEA_DTYPE_FLOAT32;
  if (cv != nullptr) {
    p.out = load_matrix(*cv, "c", dev);
    if (p.out.rows != M || p.out.cols != N)
      TB_FAIL(TRACEA_INVALID_PARAMS, "c shape [%lld,%lld] does not match expected [%lld,%lld]", p.out.rows, p.out.cols, M, N);
    check_output(p.out, "c");
    if (p.out.col_stride != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "c: the columns of a row must be contiguous");
    dtype = p.out.dtype;
  } else {
    p.out_mx = load_mx(*cq, "c_mx", dev);
    check_mx_shape(p.out_mx, "c_mx", M, N);
    p.to_mx = true;
    if (p.epi.residual) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "a residual needs a 16- or 32-bit output");
  }
  if (p.epi.residual) {
    p.residual = load_matrix(*resv, "residual", dev);
    if (p.residual.rows != M || p.residual.cols != N) TB_FAIL(TRACEA_INVALID_PARAMS, "residual shape must equal the c shape");
    if (p.residual.dtype != dtype) TB_FAIL(TRACEA_INVALID_PARAMS, "residual must have the dtype of c");
    if (p.residual.col_stride != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "residual: the columns of a row must be contiguous");
  }
  if (p.epi.bias) {
    if (biasv->rank != 1 || biasv->shape == nullptr || static_cast<long long>(biasv->shape[0]) != N)
      TB_FAIL(TRACEA_INVALID_PARAMS, "bias must have shape [%lld]", N);
    if (biasv->ptr == nullptr || biasv->device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "bias must be on device %d", dev);
    if (biasv->stride != nullptr && N > 1 && biasv->stride[0] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "bias must be contiguous");
    p.bias_is_f32 = biasv->dtype == TRACEA_DTYPE_FLOAT32;
    if (!p.bias_is_f32 && (p.to_mx || biasv->dtype != dtype))
      TB_FAIL(TRACEA_INVALID_PARAMS, "bias must be float32 or have the dtype of c");
    p.bias = biasv->ptr;
  }
  return p;
}

void mx_gemm_checked(const TraceaMxMatrix& av, const TraceaMxMatrix& wv, const TraceaTensorView* bias, const TraceaTensorView* res,
                     const TraceaTensorView* c, const TraceaMxMatrix* c_mx, const TraceaGemmParams& gp) {
  const int dev = av.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "tracea_mx_gemm takes device tensors (device_id >= 0)");
  const Mx a = load_mx(av, "a", dev);
  Product p = check_product(dev, a.rows, a.cols, wv, bias, res, c, c_mx, gp);
  p.a = a;
  if (a.rows == 0) return;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  fail_after_expired_wait(st);
  mx_product(st, p, static_cast<cudaStream_t>(gp.stream));
}

void mx_linear_checked(const TraceaTensorView& xv, const TraceaMxMatrix& wv, const TraceaTensorView* bias, const TraceaTensorView* res,
                       const TraceaTensorView* c, const TraceaMxMatrix* c_mx, const TraceaGemmParams& gp) {
  const int dev = xv.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "tracea_mx_linear takes device tensors (device_id >= 0)");
  const Matrix x = load_matrix(xv, "x", dev);
  Product p = check_product(dev, x.rows, x.cols, wv, bias, res, c, c_mx, gp);
  if (x.rows == 0) return;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  fail_after_expired_wait(st);
  const cudaStream_t stream = static_cast<cudaStream_t>(gp.stream);
  p.a.rows = x.rows;
  p.a.cols = x.cols;
  p.a.blocks = ceil_div(x.cols, tb200::kMxBlock);
  p.a.k_tiles = ceil_div(x.cols, tb200::kMxTileCols);
  const size_t data_bytes = static_cast<size_t>(x.rows * 16 * p.a.blocks + 255) / 256 * 256;
  Scratch scratch;
  scratch.alloc(st, data_bytes + static_cast<size_t>(ceil_div(x.rows, tb200::kMxTileRows) * p.a.k_tiles * tb200::kMxTileBytes), stream);
  p.a.data = static_cast<uint8_t*>(scratch.ptr);
  p.a.scales = p.a.data + data_bytes;
  quantize(x, p.a, stream);
  mx_product(st, p, stream);
}

// ------------------------------------------------------------------ norms
constexpr long long kNormMaxColumns = 16384;

tb200::NormVector load_vector(const TraceaTensorView* v, const char* name, int dev, long long C, TraceaDType dtype, bool grouped,
                              long long M, long long& groups) {
  tb200::NormVector o = {nullptr, 0, 0, 0};
  if (v == nullptr) return o;
  if (v->ptr == nullptr || v->device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be on device %d", name, dev);
  if (v->shape == nullptr || v->rank != (grouped ? 2u : 1u))
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have shape [%s%lld]", name, grouped ? "groups, " : "", C);
  const int d = grouped ? 1 : 0;
  if (static_cast<long long>(v->shape[d]) != C)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s has %llu columns, expected %lld", name, (unsigned long long)v->shape[d], C);
  if (v->stride != nullptr && C > 1 && v->stride[d] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: its columns must be contiguous", name);
  if (v->dtype != TRACEA_DTYPE_FLOAT32 && v->dtype != dtype)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be float32 or have the rows' dtype", name);
  const int es = elem_size(v->dtype);
  if ((reinterpret_cast<uintptr_t>(v->ptr) & (es - 1)) != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is not aligned to its elements", name);
  if (grouped) {
    const unsigned long long n = v->shape[0];
    if (n == 0 || n > 0x7fffffffULL || M % static_cast<long long>(n) != 0)
      TB_FAIL(TRACEA_INVALID_PARAMS, "%s has %llu groups, which do not divide the %lld rows", name, n, M);
    if (groups != 0 && n != 1 && groups != static_cast<long long>(n))
      TB_FAIL(TRACEA_INVALID_PARAMS, "%s has %llu groups, another argument has %lld", name, n, groups);
    if (n != 1) {
      groups = static_cast<long long>(n);
      o.group_stride = v->stride != nullptr ? v->stride[0] : C;
      if (o.group_stride < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: negative stride", name);
    }
  }
  o.ptr = v->ptr;
  o.f32 = v->dtype == TRACEA_DTYPE_FLOAT32 ? 1 : 0;
  o.vec = aligned16(v->ptr) && o.group_stride * es % 16 == 0 ? 1 : 0;
  return o;
}

tb200::NormStage load_stage(const TraceaNorm& n, int dev, long long C, TraceaDType dtype, long long M, long long& groups) {
  tb200::NormStage s;
  memset(&s, 0, sizeof(s));
  switch (n.kind) {
    case TRACEA_NORM_NONE: s.kind = tb200::kNormNone; break;
    case TRACEA_NORM_RMS: s.kind = tb200::kNormRms; break;
    case TRACEA_NORM_LAYER: s.kind = tb200::kNormLayer; break;
    default: TB_FAIL(TRACEA_INVALID_PARAMS, "unknown norm kind %d", static_cast<int>(n.kind));
  }
  if (!(n.eps >= 0.0f)) TB_FAIL(TRACEA_INVALID_PARAMS, "eps must not be negative");
  s.eps = n.eps;
  s.weight = load_vector(n.weight, "weight", dev, C, dtype, false, M, groups);
  s.bias = load_vector(n.bias, "bias", dev, C, dtype, false, M, groups);
  s.scale = load_vector(n.scale, "scale", dev, C, dtype, true, M, groups);
  s.shift = load_vector(n.shift, "shift", dev, C, dtype, true, M, groups);
  return s;
}

template <typename T, int kThreads, int kVecs, int kMode, bool kJoin, int kNext>
void launch_norm_kernel(const tb200::BlockNormArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int kBlock = tb200::norm_block_threads(kThreads), kRows = kBlock / kThreads;
  const long long blocks = std::min<long long>(ceil_div(a.M, kRows), static_cast<long long>(num_sms) * tb200::norm_blocks_per_sm(kThreads, kJoin));
  launch(tb200::block_norm_kernel<T, kThreads, kVecs, kMode, kJoin, kNext>, static_cast<unsigned>(blocks), kBlock, 0, 1, kLaunchNorm,
         stream, a);
}

template <typename T, int kThreads, int kVecs>
void launch_norm_shape(const tb200::BlockNormArgs& a, bool join, int next, bool vec, int num_sms, cudaStream_t stream) {
  auto go = [&](auto joined, auto nexts) {
    constexpr bool kJoin = decltype(joined)::value;
    constexpr int kNext = decltype(nexts)::value;
    constexpr int kOther = kNext == tb200::kNextMx ? tb200::kRowsSingle : tb200::kRowsSpread;
    if (vec) launch_norm_kernel<T, kThreads, kVecs, tb200::kRowsVec, kJoin, kNext>(a, num_sms, stream);
    else launch_norm_kernel<T, kThreads, kVecs, kOther, kJoin, kNext>(a, num_sms, stream);
  };
  using Rows = std::integral_constant<int, tb200::kNextRows>;
  using Quantised = std::integral_constant<int, tb200::kNextMx>;
  if (!join) {
    if (next == tb200::kNextRows) go(std::false_type{}, Rows{});
    else go(std::false_type{}, Quantised{});
  } else if (next == tb200::kNextNone) {
    go(std::true_type{}, std::integral_constant<int, tb200::kNextNone>{});
  } else if (next == tb200::kNextRows) {
    go(std::true_type{}, Rows{});
  } else {
    go(std::true_type{}, Quantised{});
  }
}

template <typename T>
void launch_norm(const tb200::BlockNormArgs& a, bool join, int next, bool vec, int num_sms, cudaStream_t stream) {
  if (a.C <= 256) launch_norm_shape<T, 32, 1>(a, join, next, vec, num_sms, stream);
  else if (a.C <= 1024) launch_norm_shape<T, 128, 1>(a, join, next, vec, num_sms, stream);
  else if (a.C <= 2048) launch_norm_shape<T, 256, 1>(a, join, next, vec, num_sms, stream);
  else if (a.C <= 4096) launch_norm_shape<T, 512, 1>(a, join, next, vec, num_sms, stream);
  else if (a.C <= 8192) launch_norm_shape<T, 1024, 1>(a, join, next, vec, num_sms, stream);
  else launch_norm_shape<T, 1024, 2>(a, join, next, vec, num_sms, stream);
}

// h == nullptr: the norm alone, of x. following == nullptr: the join alone.
void block_norm_checked(const TraceaTensorView* hv, const TraceaTensorView& xv, const TraceaNorm* join, const TraceaTensorView* gate,
                        float residual_scale, const TraceaTensorView* rv, const TraceaNorm* norm, const TraceaTensorView* yv,
                        const TraceaMxMatrix* yq, void* stream, const char* entry) {
  const int dev = xv.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s takes device tensors (device_id >= 0)", entry);
  const Matrix x = load_matrix(xv, "x", dev);
  const long long M = x.rows, C = x.cols;
  if (C == 0) TB_FAIL(TRACEA_INVALID_PARAMS, "x has no columns");
  if (C > kNormMaxColumns) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%lld columns: at most %lld", C, kNormMaxColumns);
  auto rows = [&](const TraceaTensorView& v, const char* name) {
    const Matrix m = load_matrix(v, name, dev);
    if (m.rows != M || m.cols != C)
      TB_FAIL(TRACEA_INVALID_PARAMS, "%s is [%lld,%lld], expected [%lld,%lld]", name, m.rows, m.cols, M, C);
    if (m.dtype != x.dtype) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have the dtype of x", name);
    if (m.col_stride != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: the columns of a row must be contiguous", name);
    return m;
  };
  rows(xv, "x");
  tb200::BlockNormArgs a;
  memset(&a, 0, sizeof(a));
  long long groups = 0;
  bool vec = rows_of_8(x);
  a.x = x.ptr;
  a.x_stride = x.row_stride;
  if (hv != nullptr) {
    const Matrix h = rows(*hv, "h"), r = rows(*rv, "r");
    a.h = h.ptr;
    a.h_stride = h.row_stride;
    a.r = r.ptr;
    a.r_stride = r.row_stride;
    check_output(r, "r");
    vec = vec && rows_of_8(h) && rows_of_8(r);
    a.join = load_stage(*join, dev, C, x.dtype, M, groups);
    a.gate = load_vector(gate, "gate", dev, C, x.dtype, true, M, groups);
    a.residual_scale = residual_scale;
  }
  int next = tb200::kNextNone;
  if (norm != nullptr) {
    if ((yv == nullptr) == (yq == nullptr)) TB_FAIL(TRACEA_INVALID_PARAMS, "exactly one of y and y_mx must be given");
    a.norm = load_stage(*norm, dev, C, x.dtype, M, groups);
    if (yv != nullptr) {
      const Matrix y = rows(*yv, "y");
      a.y = y.ptr;
      a.y_stride = y.row_stride;
      check_output(y, "y");
      vec = vec && rows_of_8(y);
      next = tb200::kNextRows;
    } else {
      const Mx q = load_mx(*yq, "y_mx", dev);
      check_mx_shape(q, "y_mx", M, C);
      a.codes = q.data;
      a.scales = q.scales;
      a.blocks = static_cast<int>(q.blocks);
      a.k_tiles = static_cast<int>(q.k_tiles);
      next = tb200::kNextMx;
    }
  } else if (yv != nullptr || yq != nullptr) {
    TB_FAIL(TRACEA_INVALID_PARAMS, "y is given without the norm that makes it");
  }
  if (M == 0) return;
  a.M = M;
  a.C = static_cast<int>(C);
  a.rows_per_group = groups > 0 ? M / groups : 0;
  vec = vec && C % 8 == 0;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  by_dtype(x.dtype, [&](auto tag) {
    launch_norm<decltype(tag)>(a, hv != nullptr, next, vec, st.num_sms, static_cast<cudaStream_t>(stream));
  });
}

}  // namespace

// ==================================================================== exported C ABI
extern "C" {

uint64_t tracea_mx_data_bytes(uint64_t rows, uint64_t cols) {
  if (rows > 0x7fffffffULL || cols > 0x7fffff00ULL) return 0;
  return rows * 16u * ((cols + 31u) / 32u);
}
uint64_t tracea_mx_scale_bytes(uint64_t rows, uint64_t cols) {
  if (rows > 0x7fffffffULL || cols > 0x7fffff00ULL) return 0;
  return ((rows + 127u) / 128u) * ((cols + 127u) / 128u) * 512u;
}

TraceaStatus tracea_mx_quantize(TraceaTensorView x, TraceaMxMatrix* q, void* stream) {
  return guarded("tracea_mx_quantize", [&] { mx_quantize_checked(x, q, stream); });
}
TraceaStatus tracea_mx_dequantize(TraceaMxMatrix q, TraceaTensorView* out, void* stream) {
  return guarded("tracea_mx_dequantize", [&] { mx_dequantize_checked(q, out, stream); });
}
TraceaStatus tracea_mx_gemm(TraceaMxMatrix a, TraceaMxMatrix w, const TraceaTensorView* bias, const TraceaTensorView* residual,
                            TraceaTensorView* c, TraceaMxMatrix* c_mx, TraceaGemmParams params) {
  return guarded("tracea_mx_gemm", [&] { mx_gemm_checked(a, w, bias, residual, c, c_mx, params); });
}
TraceaStatus tracea_mx_linear(TraceaTensorView x, TraceaMxMatrix w, const TraceaTensorView* bias, const TraceaTensorView* residual,
                              TraceaTensorView* c, TraceaMxMatrix* c_mx, TraceaGemmParams params) {
  return guarded("tracea_mx_linear", [&] { mx_linear_checked(x, w, bias, residual, c, c_mx, params); });
}
TraceaStatus tracea_block_norm(TraceaTensorView x, const TraceaNorm* norm, TraceaTensorView* y, TraceaMxMatrix* y_mx, void* stream) {
  return guarded("tracea_block_norm", [&] {
    if (norm == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "Null pointer in norm arguments");
    block_norm_checked(nullptr, x, nullptr, nullptr, 0.0f, nullptr, norm, y, y_mx, stream, "tracea_block_norm");
  });
}
TraceaStatus tracea_block_norm_add(TraceaTensorView h, TraceaTensorView x, const TraceaNorm* norm, const TraceaTensorView* gate,
                                   float residual_scale, TraceaTensorView* r, const TraceaNorm* following, TraceaTensorView* y,
                                   TraceaMxMatrix* y_mx, void* stream) {
  return guarded("tracea_block_norm_add", [&] {
    if (norm == nullptr || r == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "Null pointer in norm arguments");
    block_norm_checked(&h, x, norm, gate, residual_scale, r, following, y, y_mx, stream, "tracea_block_norm_add");
  });
}

}  // extern "C"
