// Host side of the norms around a block: tracea_block_norm, tracea_block_norm_add. The reference has no counterpart.
#include "mx_host.cuh"
#include "block_norm_sm100.cuh"

namespace {

using namespace tb200_host;

constexpr long long kNormMaxColumns = 16384;

tb200::NormVector load_vector(const TraceaTensorView* v, const char* name, int dev, long long C, TraceaDType dtype, bool grouped,
                              long long M, long long& groups) {
  tb200::NormVector o = {nullptr, 0, 0, 0};
  if (v == nullptr) return o;
  const bool none = grouped && M == 0;                              // no samples, and so maybe no groups
  if ((v->ptr == nullptr && !none) || v->device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be on device %d", name, dev);
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
    if (none) return o;
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
void launch_norm_kernel(const tb200::BlockNormArgs& a, int dev, int num_sms, cudaStream_t stream) {
  constexpr int kBlock = tb200::norm_block_threads(kThreads, kVecs, kJoin);
  const long long blocks =
      std::min<long long>(a.M, static_cast<long long>(num_sms) * tb200::norm_blocks_per_sm(kThreads, kVecs, kJoin, sizeof(T)));
  constexpr int kSmem = tb200::norm_smem_bytes(kThreads, kVecs, kMode, kJoin, kNext, sizeof(T));
  auto kern = tb200::block_norm_kernel<T, kThreads, kVecs, kMode, kJoin, kNext>;
  if constexpr (kSmem > 47 * 1024) {
    static std::atomic<bool> done[kMaxDevices];
    if (!done[dev].load(std::memory_order_relaxed)) {
      TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
      done[dev].store(true, std::memory_order_relaxed);
    }
  }
  launch(kern, static_cast<unsigned>(blocks), kBlock, kSmem, 1, kLaunchNorm, stream, a);
}

template <typename T, int kThreads, int kVecs, bool kVecOnly = false>
void launch_norm_shape(const tb200::BlockNormArgs& a, bool join, int next, bool vec, int dev, int num_sms, cudaStream_t stream) {
  auto go = [&](auto joined, auto nexts) {
    constexpr bool kJoin = decltype(joined)::value;
    constexpr int kNext = decltype(nexts)::value;
    constexpr int kOther = kNext == tb200::kNextMx ? tb200::kRowsSingle : tb200::kRowsSpread;
    if (kVecOnly || vec) launch_norm_kernel<T, kThreads, kVecs, tb200::kRowsVec, kJoin, kNext>(a, dev, num_sms, stream);
    else if constexpr (!kVecOnly) launch_norm_kernel<T, kThreads, kVecs, kOther, kJoin, kNext>(a, dev, num_sms, stream);
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
void launch_norm(const tb200::BlockNormArgs& a, bool join, int next, bool vec, int dev, int num_sms, cudaStream_t stream) {
  // A warp to a row of up to 1024 columns, or two. One costs fewer instructions, two have more rows' loads under way. Layer norm,
  // the same quantised, its join, with the next norm, with that quantised, us, two warps / one, 1024 columns of bf16:
  //     148 rows  2.8 2.9   3.0 3.3   2.8 2.9   3.4 3.5   3.7 4.0        20000 rows  17 16   21 19   20 20   31 29    34 28
  //   12544 rows   13 11    14 12     14 12     21 17     23 20          80000 rows  58 61   68 58   86 81  116 117  117 88
  // 704 of fp32, 12544 rows: 17 15, 17 16, 20 18, 29 26, 29 26; 80000: 81 79, 75 70, 108 122, 151 165, 152 122. Rows that are not
  // 16-byte aligned lose as often as they win. The choice may depend on the rows alone, not on what the call does with them:
  // aligned alike, the same rows have the same bits in all of a call's forms. (The bound on bytes is the fp32 rows'; 16-bit ones past it
  // would gain in three forms and lose up to 5 % in two.)
  const bool warp_rows = vec && a.M >= 4 * num_sms && static_cast<long long>(a.M) * a.C * static_cast<long long>(sizeof(T)) <= (40LL << 20);
  if (a.C <= 256) launch_norm_shape<T, 32, 1>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 512) launch_norm_shape<T, 32, 2>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 1024 && warp_rows) launch_norm_shape<T, 32, 4, true>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 1024) launch_norm_shape<T, 64, 2>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 2048) launch_norm_shape<T, 128, 2>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 4096) launch_norm_shape<T, 256, 2>(a, join, next, vec, dev, num_sms, stream);
  else if (a.C <= 8192) launch_norm_shape<T, 512, 2>(a, join, next, vec, dev, num_sms, stream);
  else launch_norm_shape<T, 512, 4>(a, join, next, vec, dev, num_sms, stream);
}

// h == nullptr: the norm alone, of x. following == nullptr: the join alone.
void block_norm_checked(const TraceaTensorView* hv, const TraceaTensorView& xv, const TraceaNorm* join, const TraceaTensorView* gate,
                        float residual_scale, const TraceaTensorView* rv, const TraceaNorm* norm, const TraceaTensorView* yv,
                        const TraceaMxMatrix* yq, void* stream, const char* entry) {
  const int dev = xv.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s takes device tensors (device_id >= 0)", entry);
  const Matrix x = load_matrix(xv, "x", dev);
  check_rows(x, "x");
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
  a.M = static_cast<int>(M);
  a.C = static_cast<int>(C);
  a.rows_per_group = groups > 0 ? static_cast<int>(M / groups) : 0;
  vec = vec && C % 8 == 0;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  by_dtype(x.dtype, [&](auto tag) {
    launch_norm<decltype(tag)>(a, hv != nullptr, next, vec, dev, st.num_sms, static_cast<cudaStream_t>(stream));
  });
}

}  // namespace

// ==================================================================== exported C ABI
extern "C" {

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
