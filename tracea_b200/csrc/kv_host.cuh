// Host helpers of the operators on rows of heads and on the cache of keys and values: their views and their checks.
#pragma once
#include "heads_sm100.cuh"
#include "mx_host.cuh"

namespace __attribute__((visibility("hidden"))) tb200_host {

// ------------------------------------------------------------------ views
struct Heads {
  char* ptr;
  long long tokens, heads, cols, token_stride, head_stride;   // strides in elements; columns are contiguous
  TraceaDType dtype;
  int es;
  bool vec;                                                   // every head starts on a 16-byte boundary
};

inline Heads load_heads(const TraceaTensorView& v, const char* name, int dev) {
  if (v.rank != 3 || v.shape == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have shape [tokens, heads, columns]", name);
  Heads h;
  for (int i = 0; i < 3; ++i)
    if (v.shape[i] > 0x7fffff00ULL) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: shape[%d] = %llu is out of range", name, i, (unsigned long long)v.shape[i]);
  h.ptr = static_cast<char*>(v.ptr);
  h.tokens = static_cast<long long>(v.shape[0]);
  h.heads = static_cast<long long>(v.shape[1]);
  h.cols = static_cast<long long>(v.shape[2]);
  if (h.heads == 0 || h.cols == 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s has no %s", name, h.heads == 0 ? "heads" : "columns");
  h.dtype = v.dtype;
  h.es = elem_size(v.dtype);
  if (h.es == 0) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: unsupported dtype %s", name, dtype_name(v.dtype));
  if (v.device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is on device %d, expected %d", name, v.device_id, dev);
  if (h.tokens > 0 && v.ptr == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s has a NULL pointer", name);
  if ((reinterpret_cast<uintptr_t>(v.ptr) & (h.es - 1)) != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is not aligned to its elements", name);
  if (v.stride != nullptr && h.cols > 1 && v.stride[2] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s: a head's columns must be contiguous", name);
  h.token_stride = v.stride != nullptr && h.tokens > 1 ? v.stride[0] : h.heads * h.cols;
  h.head_stride = v.stride != nullptr && h.heads > 1 ? v.stride[1] : h.cols;
  if (h.token_stride < 0 || h.head_stride < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s: negative stride", name);
  h.vec = aligned16(h.ptr) && h.token_stride * h.es % 16 == 0 && h.head_stride * h.es % 16 == 0;
  return h;
}

inline void check_heads_output(const Heads& h, const char* name) {
  const bool tokens_apart = h.tokens <= 1 || h.token_stride >= (h.heads - 1) * h.head_stride + h.cols;
  const bool heads_apart = h.heads <= 1 || h.head_stride >= (h.tokens - 1) * h.token_stride + h.cols;
  if (!((tokens_apart && (h.heads <= 1 || h.head_stride >= h.cols)) || (heads_apart && (h.tokens <= 1 || h.token_stride >= h.cols))))
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s: its rows overlap", name);
}

inline void check_like(const Heads& h, const char* name, const Heads& x, const char* other) {
  if (h.tokens != x.tokens || h.cols != x.cols)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s has %lld tokens of %lld columns, %s has %lld of %lld", name, h.tokens, h.cols, other, x.tokens, x.cols);
  if (h.dtype != x.dtype) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have the dtype of %s", name, other);
}

// A vector over a head's columns.
inline const void* load_head_weight(const TraceaTensorView* v, const char* name, int dev, long long cols, TraceaDType dtype, int& f32) {
  f32 = 0;
  if (v == nullptr) return nullptr;
  if (v->rank != 1 || v->shape == nullptr || static_cast<long long>(v->shape[0]) != cols)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have shape [%lld]", name, cols);
  if (v->ptr == nullptr || v->device_id != dev) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be on device %d", name, dev);
  if (v->stride != nullptr && cols > 1 && v->stride[0] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s must be contiguous", name);
  if (v->dtype != TRACEA_DTYPE_FLOAT32 && v->dtype != dtype)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be float32 or have the rows' dtype", name);
  if ((reinterpret_cast<uintptr_t>(v->ptr) & (elem_size(v->dtype) - 1)) != 0)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%s is not aligned to its elements", name);
  f32 = v->dtype == TRACEA_DTYPE_FLOAT32 ? 1 : 0;
  return v->ptr;
}

inline tb200::HeadRows load_head_rows(const Heads& x, const Heads* y, const void* weight, int weight_f32) {
  tb200::HeadRows r;
  memset(&r, 0, sizeof(r));
  r.x = x.ptr;
  r.weight = weight;
  r.weight_f32 = weight_f32;
  r.heads = static_cast<int>(x.heads);
  r.x_token = x.token_stride;
  r.x_head = x.head_stride;
  if (y != nullptr) {
    r.y = y->ptr;
    r.y_token = y->token_stride;
    r.y_head = y->head_stride;
  }
  return r;
}

inline tb200::Rotation load_rotation(const TraceaRotation* v, long long cols) {
  tb200::Rotation r = {nullptr, 0, 0};
  if (v == nullptr || v->pairs == 0) return r;
  if (v->frequencies == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "the rotation has no frequencies");
  if ((reinterpret_cast<uintptr_t>(v->frequencies) & 7u) != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "the frequencies are not aligned to their elements");
  if (2 * static_cast<long long>(v->pairs) > cols)
    TB_FAIL(TRACEA_INVALID_PARAMS, "%u pairs of columns to rotate, of %lld columns", v->pairs, cols);
  r.frequencies = v->frequencies;
  r.pairs = static_cast<int>(v->pairs);
  r.interleaved = v->interleaved != 0 ? 1 : 0;
  return r;
}

inline int load_head_norm(TraceaNormKind kind, float eps) {
  if (kind != TRACEA_NORM_NONE && kind != TRACEA_NORM_RMS) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "norm kind %d: heads have none or rms", static_cast<int>(kind));
  if (!(eps >= 0.0f)) TB_FAIL(TRACEA_INVALID_PARAMS, "eps must not be negative");
  return kind == TRACEA_NORM_RMS ? 1 : 0;
}

// Lanes that hold a row, 16 columns each.
inline int head_lanes(long long cols) {
  int lanes = 1;
  while (lanes * 16 < cols) lanes *= 2;
  return lanes;
}

inline tb200::CacheRef load_cache(const TraceaKvCache& c) {
  tb200::CacheRef r;
  memset(&r, 0, sizeof(r));
  if (c.device_id < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "the cache must be in device memory");
  if (c.pages > 0x7fffffffULL || c.heads == 0 || c.heads > 0xffffu) TB_FAIL(TRACEA_INVALID_PARAMS, "cache: %llu pages of %u heads are out of range", (unsigned long long)c.pages, c.heads);
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
    TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "cache: pages of %u tokens: 16, 32, 64 or 128", c.page_size);
  if (c.head_dim == 0 || c.head_dim % 16 != 0 || c.head_dim > tb200::kCacheMaxColumns)
    TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "cache: heads of %u columns: a multiple of 16 up to %d", c.head_dim, tb200::kCacheMaxColumns);
  if (c.pages > 0 && (c.k == nullptr || c.v == nullptr || c.k_scales == nullptr || c.v_scales == nullptr))
    TB_FAIL(TRACEA_INVALID_PARAMS, "the cache has a NULL pointer");
  if (!aligned16(c.k) || !aligned16(c.v)) TB_FAIL(TRACEA_INVALID_PARAMS, "cache: keys and values must be 16-byte aligned");
  r.k = static_cast<uint8_t*>(c.k);
  r.v = static_cast<uint8_t*>(c.v);
  r.k_scales = c.k_scales;
  r.v_scales = c.v_scales;
  r.pages = static_cast<long long>(c.pages);
  r.heads = static_cast<int>(c.heads);
  r.D = static_cast<int>(c.head_dim);
  for (r.page_shift = 4; (1u << r.page_shift) != c.page_size; ++r.page_shift) {}
  return r;
}

inline void check_int_vector(const TraceaTensorView& v, const char* name, int dev, long long n) {
  if (v.rank != 1 || v.shape == nullptr || static_cast<long long>(v.shape[0]) != n) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must have shape [%lld]", name, n);
  if (v.dtype != TRACEA_DTYPE_INT32) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be int32", name);
  if (v.stride != nullptr && n > 1 && v.stride[0] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%s must be contiguous", name);
  if (n > 0 && (v.ptr == nullptr || v.device_id != dev)) TB_FAIL(TRACEA_INVALID_PARAMS, "%s must be on device %d", name, dev);
  if ((reinterpret_cast<uintptr_t>(v.ptr) & 3u) != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%s is not aligned to its elements", name);
}

inline tb200::SequencesRef load_sequences(const TraceaSequences& s, int dev, long long rows) {
  tb200::SequencesRef r;
  memset(&r, 0, sizeof(r));
  const TraceaTensorView& t = s.pages;
  if (t.rank != 2 || t.shape == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "pages must have shape [sequences, pages]");
  if (t.shape[0] > 0x7fffff00ULL || t.shape[1] > 0x7fffffULL) TB_FAIL(TRACEA_INVALID_PARAMS, "pages is out of range");
  if (t.dtype != TRACEA_DTYPE_INT32) TB_FAIL(TRACEA_INVALID_PARAMS, "pages must be int32");
  const long long n = static_cast<long long>(t.shape[0]), width = static_cast<long long>(t.shape[1]);
  if (t.stride != nullptr && width > 1 && t.stride[1] != 1) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "pages: a sequence's entries must be contiguous");
  r.table_stride = t.stride != nullptr && n > 1 ? t.stride[0] : width;
  if (r.table_stride < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "pages: negative stride");
  if (n > 0 && width > 0 && (t.ptr == nullptr || t.device_id != dev)) TB_FAIL(TRACEA_INVALID_PARAMS, "pages must be on device %d", dev);
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 3u) != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "pages is not aligned to its elements");
  check_int_vector(s.lengths, "lengths", dev, n);
  if (s.starts != nullptr) {
    check_int_vector(*s.starts, "starts", dev, n + 1);
    r.starts = static_cast<const int*>(s.starts->ptr);
  } else if (rows != n) {
    TB_FAIL(TRACEA_INVALID_PARAMS, "%lld rows of %lld sequences, of which each has one where starts is not given", rows, n);
  }
  r.table = static_cast<const int*>(t.ptr);
  r.lengths = static_cast<const int*>(s.lengths.ptr);
  r.table_width = static_cast<int>(width);
  r.count = static_cast<int>(n);
  r.rows = static_cast<int>(rows);
  return r;
}

}  // namespace tb200_host
