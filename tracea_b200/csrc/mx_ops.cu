// Host side of the 4-bit microscaled operators: tracea_mx_quantize, tracea_mx_dequantize, tracea_mx_gemm, tracea_mx_linear. The
// reference has no counterpart of any of them.
#include "mx_host.cuh"
#include "mx_gemm_sm100.cuh"
#include "mx_tokens_sm100.cuh"

namespace {

using namespace tb200_host;

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

std::atomic<bool> g_mx_attr_set[kMaxDevices][3][4][3];

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
  constexpr int stages = tb200::mx_num_stages(BN, kPair, kStore), smem = tb200::mx_smem_bytes(BN, stages, kPair, kStore);
  static_assert(!kPair || smem >= tb200::kPairMinSmem, "see there");
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
  launch(kern, grid_of(kPair ? 2 * workers : workers), tb200::mx_threads(BN, kPair, kStore), smem, kPair ? 2 : 1,
         kLaunchMxGemm, stream, ta, tw, tsa, tsw, to, g);
}

// ------------------------------------------------------------------ few rows
struct TokensPlan {
  int cols = 0, split = 1, steps = 0, stages = 0;   // cols == 0: not for this problem
  bool fused = false;
};

// `in_place`: x is at hand in its storage type, its columns contiguous. The form of few rows, and quantising inside it, where they are
// the faster ones (us, rows / this form / the general one):
//   4096 x 4096   1 4.8 7.6   32 5.5 7.4   64 6.6 7.1  128 7.3 7.2        1000 x 2048    1 3.6 4.9   32 4.3 5.0  64 5.0 5.0  128 6.7 5.2
//   4096 x 1024   1 3.6 4.2   32 4.0 4.2   64 4.6 4.1  128 6.2 4.2        256 x 16384    1 4.2 18   128 7.3 18
// Quantising inside costs each CTA rows x steps passes of eight warps, a launch and a round trip ~2.2 us.
TokensPlan plan_tokens(long long M, long long N, long long K, bool to_mx, bool in_place, int num_sms) {
  TokensPlan p;
  static const int knob_rows = env_int("TRACEA_B200_MX_TOKENS", tb200::kTokMaxRows);
  static const int knob_fused = env_int("TRACEA_B200_MX_FUSED", 64);
  const long long n_tiles = ceil_div(N, 128), k_iters = ceil_div(K, 256), m_tiles = ceil_div(M, tb200::kTokMaxRows);
  if (knob_rows == 0 || (M > 64 && m_tiles * n_tiles > num_sms)) return p;
  int split = 1;
  while (split < (to_mx ? 4 : 8) && 2 * split <= k_iters && m_tiles * n_tiles * 2 * split <= num_sms) split *= 2;
  if (!(M <= 32 || (M <= 64 && k_iters >= 8) || (split > 1 && k_iters >= 16))) return p;
  p.cols = static_cast<int>(ceil_div(std::min<long long>(M, tb200::kTokMaxRows), 16) * 16);
  p.split = split;
  p.steps = static_cast<int>(ceil_div(k_iters, split));
  p.fused = in_place && M <= 16 && M * p.steps <= knob_fused && p.steps <= tb200::kTokFusedSteps;
  // more CTAs than SMs: two to an SM
  const int share = m_tiles * n_tiles * split > num_sms ? 232448 / 2 - 1024 : 232448;
  const int room = share - 1024 - tb200::kTokBarrierBytes - (p.fused ? p.steps * static_cast<int>(tb200::tok_step_bytes(p.cols)) : 0);
  const int stage = static_cast<int>(tb200::kTokWBytes + (p.fused ? 0u : tb200::tok_step_bytes(p.cols)));
  p.stages = std::max(1, std::min({p.steps, tb200::kTokMaxStages, room / stage}));
  return p;
}

template <typename OutT, typename InT, bool kFused, bool kMxOut>
void launch_tokens(DeviceState& st, const Product& p, const Matrix* x, const TokensPlan& plan, cudaStream_t stream) {
  auto kern = tb200::mx_tokens_sm100_kernel<OutT, InT, kFused, kMxOut>;
  static std::atomic<bool> done[kMaxDevices];
  if (!done[st.dev].load(std::memory_order_relaxed)) {
    TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
    done[st.dev].store(true, std::memory_order_relaxed);
  }
  tb200::MxTokensArgs g;
  memset(&g, 0, sizeof(g));
  g.M = static_cast<int>(p.a.rows);
  g.N = static_cast<int>(p.w.rows);
  g.K = static_cast<int>(p.a.cols);
  g.cols = plan.cols;
  g.k_iters = static_cast<int>(ceil_div(p.a.cols, 256));
  g.split = plan.split;
  g.num_stages = plan.stages;
  g.idesc = tb200::ptx::make_mx_idesc(128, static_cast<uint32_t>(plan.cols));
  CUtensorMap tw, tsw, ta, tsa;
  encode_codes(&tw, p.w, 128);
  encode_scales(&tsw, p.w, 1);
  if constexpr (kFused) {
    memset(&ta, 0, sizeof(ta));
    memset(&tsa, 0, sizeof(tsa));
    g.x = x->ptr;
    g.x_stride = x->row_stride;
    g.x_vec = rows_of_8(*x) ? 1 : 0;
  } else {
    encode_codes(&ta, p.a, plan.cols);
    encode_scales(&tsa, p.a, 1);
  }
  if constexpr (kMxOut) {
    g.out = p.out_mx.data;
    g.out_scales = p.out_mx.scales;
    g.out_blocks = static_cast<int>(p.out_mx.blocks);
    g.out_k_tiles = static_cast<int>(p.out_mx.k_tiles);
  } else {
    g.out = p.out.ptr;
    g.out_stride = p.out.row_stride;
    g.out_vec = reinterpret_cast<uintptr_t>(p.out.ptr) % (4 * sizeof(OutT)) == 0 && p.out.row_stride % 4 == 0 ? 1 : 0;
    if (p.epi.residual) {
      g.residual = p.residual.ptr;
      g.res_stride = p.residual.row_stride;
    }
  }
  g.bias = p.bias;
  g.bias_is_f32 = p.bias_is_f32 ? 1 : 0;
  g.act = p.epi.act;
  g.status = st.status;
  const long long limit = g_test_wait_limit.load(std::memory_order_relaxed);
  g.wait_limit = limit > 0 ? limit : tb200::kWaitLimitCycles;
  g.test_producer_stop = g_test_producer_stop.load(std::memory_order_relaxed);
  launch(kern, dim3(grid_of(ceil_div(p.w.rows, 128) * plan.split), grid_of(ceil_div(p.a.rows, tb200::kTokMaxRows))), tb200::kTokThreads,
         tb200::tok_smem_bytes(plan.cols, plan.stages, kFused ? plan.steps : 0), plan.split, kLaunchMxTokens, stream, tw, tsw, ta, tsa, g);
}

void tokens_product(DeviceState& st, const Product& p, const Matrix* x, const TokensPlan& plan, cudaStream_t stream) {
  if (p.to_mx) {
    if (plan.fused)
      by_dtype(x->dtype, [&](auto tag) { launch_tokens<__nv_bfloat16, decltype(tag), true, true>(st, p, x, plan, stream); });
    else
      launch_tokens<__nv_bfloat16, float, false, true>(st, p, x, plan, stream);
    return;
  }
  by_dtype(p.out.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (plan.fused) launch_tokens<T, T, true, false>(st, p, x, plan, stream);
    else launch_tokens<T, float, false, false>(st, p, x, plan, stream);
  });
}

// Columns of a tile: 64 or 128 in a CTA, 192 or 256 in a pair of CTAs (256 rows). By the time of the busiest CTA or pair, in
// us: what a launch takes once, and per wave of tiles either its k-steps (an SM has 16 KB of A and half or all of the columns' rows
// of W to bring in a step) and what lies between two tiles, or its epilogue, whichever is longer. 192 columns have two accumulators,
// 256 one, which pays for its wider steps only over a long K. Measured / this formula, columns 64, 128, 192, 256, bf16 outputs (fp32 and
// 4-bit ones take the same choice):
//   8192 x 8192 x 8192         352 251 204 192 / 444 261 212 206     12544 x 4096 x 1024    49  38  31 34 / 53 33 31 36
//   4096 x 4096 x 4096          49  32  30  32 / 59  36  32  35      the same, SiLU          53  41  41 47 / 53 41 42 47
//   2048 x 2048 x 2048        12.6 7.3 9.2 9.1 / 11 7.9 10 8.7       1024 x 1024 x 2048   4.8 5.3 6.7  - / 4.8 5.4 7.0 8.6
int pick_mx_tile(long long M, long long N, long long K, int act, int num_sms) {
  static const int forced = env_int("TRACEA_B200_MX_BN", 0);
  if (forced != 0) return forced;
  struct Form {
    int bn;
    double once, step, between, epilogue, epilogue_act;
  };
  static const Form forms[4] = {{64, 2.6, 0.24, 0.2, 0.75, 0.9}, {128, 2.9, 0.28, 0.25, 1.15, 1.75},
                                {192, 4.0, 0.33, 0.4, 1.8, 2.5}, {256, 4.0, 0.41, 1.3, 2.7, 3.9}};
  const double steps = static_cast<double>(ceil_div(K, 256));
  int best = 0;
  double best_time = 0.0;
  for (const Form& f : forms) {
    const bool pair = f.bn >= 192;
    const long long waves = ceil_div(ceil_div(M, pair ? 256 : 128) * ceil_div(N, f.bn), pair ? num_sms / 2 : num_sms);
    const double epilogue = act == tb200::kActSilu || act == tb200::kActGelu ? f.epilogue_act : f.epilogue;
    const double time = f.once + static_cast<double>(waves) * std::max(steps * f.step + f.between, epilogue);
    if (best == 0 || time < best_time) {
      best = f.bn;
      best_time = time;
    }
  }
  return best;
}

void mx_product(DeviceState& st, const Product& p, cudaStream_t stream) {
  const TokensPlan plan = plan_tokens(p.a.rows, p.w.rows, p.a.cols, p.to_mx, false, st.num_sms);
  if (plan.cols != 0) {
    tokens_product(st, p, nullptr, plan, stream);
    return;
  }
  const int bn = pick_mx_tile(p.a.rows, p.w.rows, p.a.cols, p.epi.act, st.num_sms);
  auto tiled = [&](auto tag, int dt, auto store) {
    using T = decltype(tag);
    constexpr int kStore = decltype(store)::value;
    if (bn == 256) launch_mx_gemm<T, 256, true, kStore>(st, dt, p, stream);
    else if (bn == 192) launch_mx_gemm<T, 192, true, kStore>(st, dt, p, stream);
    else if (bn == 128) launch_mx_gemm<T, 128, false, kStore>(st, dt, p, stream);
    else launch_mx_gemm<T, 64, false, kStore>(st, dt, p, stream);
  };
  if (p.to_mx) {
    tiled(__nv_bfloat16{}, 0, std::integral_constant<int, tb200::kMxStoreMx>{});
    return;
  }
  // (a store that ends inside 16 bytes would write all of them, past a row's end where its stride leaves room)
  const bool tma = aligned16(p.out.ptr) && p.out.row_stride * p.out.es % 16 == 0 && p.out.cols * p.out.es % 16 == 0;
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
    if ((reinterpret_cast<uintptr_t>(biasv->ptr) & (elem_size(biasv->dtype) - 1)) != 0)
      TB_FAIL(TRACEA_INVALID_PARAMS, "bias is not aligned to its elements");
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
  check_rows(x, "x");
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
  const bool in_place = x.col_stride == 1 && (p.to_mx || x.dtype == p.out.dtype);
  const TokensPlan plan = plan_tokens(x.rows, p.w.rows, x.cols, p.to_mx, in_place, st.num_sms);
  if (plan.fused) {
    tokens_product(st, p, &x, plan, stream);
    return;
  }
  const size_t data_bytes = static_cast<size_t>(x.rows * 16 * p.a.blocks + 255) / 256 * 256;
  Scratch scratch;
  scratch.alloc(st, data_bytes + static_cast<size_t>(ceil_div(x.rows, tb200::kMxTileRows) * p.a.k_tiles * tb200::kMxTileBytes), stream);
  p.a.data = static_cast<uint8_t*>(scratch.ptr);
  p.a.scales = p.a.data + data_bytes;
  quantize(x, p.a, stream);
  mx_product(st, p, stream);
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
}  // extern "C"
