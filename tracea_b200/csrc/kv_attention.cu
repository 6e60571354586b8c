// Host side of attention over the cache of keys and values: tracea_kv_attention. The reference has no counterpart.
#include "kv_host.cuh"
#include "kv_rows_sm100.cuh"
#include "kv_tokens_sm100.cuh"

namespace {

using namespace tb200_host;

template <typename T, int kD>
void launch_tokens(const tb200::KvAttentionArgs& a, int splits, int dev, cudaStream_t stream) {
  constexpr int kSmem = tb200::kv_token_smem_bytes<kD>();
  auto kern = tb200::kv_tokens_kernel<T, kD>;
  static std::atomic<bool> done[kMaxDevices];
  if (!done[dev].load(std::memory_order_relaxed)) {
    TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    done[dev].store(true, std::memory_order_relaxed);
  }
  const long long heads = static_cast<long long>(a.cache.heads) * a.row_tiles;
  if (heads > 65535) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%d heads of keys with %d tiles of rows", a.cache.heads, a.row_tiles);
  const dim3 grid(grid_of(static_cast<long long>(a.seqs.count) * splits), static_cast<unsigned>(heads));
  launch(kern, grid, tb200::kKvTokenThreads, kSmem, splits, kLaunchKvTokens, stream, a);
}

template <typename T, int kD>
void launch_rows(const tb200::KvAttentionArgs& a, long long items, int dev, cudaStream_t stream) {
  constexpr int kSmem = tb200::kv_rows_smem_bytes<kD>();
  auto kern = tb200::kv_rows_kernel<T, kD>;
  static std::atomic<bool> done[kMaxDevices];
  if (!done[dev].load(std::memory_order_relaxed)) {
    cudaFuncAttributes attr;
    TB_CUDA(cudaFuncGetAttributes(&attr, kern));
    if (attr.numRegs < 128) TB_FAIL(TRACEA_UNKNOWN_ERROR, "the kernel was built with too few registers to be split");   // its warps would wait for them
    TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    done[dev].store(true, std::memory_order_relaxed);
  }
  launch(kern, grid_of(items * a.cache.heads), tb200::kKvRowsThreads, kSmem, 1, kLaunchKvRows, stream, a);
}

template <typename F>
void by_half_dtype(TraceaDType t, F&& f) {
  if (t == TRACEA_DTYPE_BFLOAT16) f(__nv_bfloat16{});
  else f(__half{});
}

void kv_attention_checked(const TraceaTensorView& qv, const TraceaKvCache& cache, const TraceaSequences& seqs, const TraceaTensorView* ov,
                          const TraceaKvAttentionParams& params) {
  if (ov == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "Null pointer in attention arguments");
  tb200::KvAttentionArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = load_cache(cache);
  const int dev = cache.device_id;
  const Heads q = load_heads(qv, "q", dev), out = load_heads(*ov, "out", dev);
  if (q.dtype != TRACEA_DTYPE_BFLOAT16 && q.dtype != TRACEA_DTYPE_FLOAT16)
    TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "q must be float16 or bfloat16, not %s", dtype_name(q.dtype));
  check_like(out, "out", q, "q");
  if (out.heads != q.heads) TB_FAIL(TRACEA_INVALID_PARAMS, "out has %lld heads, q has %lld", out.heads, q.heads);
  check_heads_output(out, "out");
  if (q.cols != a.cache.D || q.heads % a.cache.heads != 0)
    TB_FAIL(TRACEA_INVALID_PARAMS, "q has %lld heads of %lld columns, the cache %d of %d", q.heads, q.cols, a.cache.heads, a.cache.D);
  if (!(params.scale > -INFINITY && params.scale < INFINITY)) TB_FAIL(TRACEA_INVALID_PARAMS, "scale must be finite");
  if (params.window > 0x7fffffffu) TB_FAIL(TRACEA_INVALID_PARAMS, "window is out of range");
  a.seqs = load_sequences(seqs, dev, q.tokens);
  if (q.tokens * (q.heads / a.cache.heads) > 0x7fffff00LL) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "q: too many rows");
  if (q.tokens == 0 || a.seqs.count == 0) return;
  a.q = q.ptr;
  a.out = out.ptr;
  a.q_token = q.token_stride;
  a.q_head = q.head_stride;
  a.out_token = out.token_stride;
  a.out_head = out.head_stride;
  a.q_vec = q.vec ? 1 : 0;
  a.out_vec = out.vec ? 8 : (reinterpret_cast<uintptr_t>(out.ptr) & 7u) == 0 && out.token_stride % 4 == 0 && out.head_stride % 4 == 0 ? 4 : 1;
  a.group = static_cast<int>(q.heads / a.cache.heads);
  a.causal = params.causal != 0 ? 1 : 0;
  a.window = static_cast<int>(std::min(params.window, 0x40000000u));   // no sequence is longer
  a.scale_log2 = fabsf(params.scale) * 1.4426950408889634f;
  a.sign = params.scale < 0.0f ? -1.0f : 1.0f;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  const cudaStream_t stream = static_cast<cudaStream_t>(params.stream);
  fail_after_expired_wait(st);
  a.status = st.status;
  const long long limit = g_test_wait_limit.load(std::memory_order_relaxed);
  a.wait_limit = limit > 0 ? limit : tb200::kWaitLimitCycles;
  a.test_producer_stop = g_test_producer_stop.load(std::memory_order_relaxed);

  // Which kernel takes a sequence depends on its rows alone, which the host does not know: it leaves out a kernel that could have none.
  const long long all_rows = q.tokens * a.group;
  constexpr int kFew = tb200::kKvTokenRows * tb200::kKvTokenTiles;
  const bool only_few = a.seqs.starts == nullptr || all_rows <= kFew, only_many = !only_few && a.seqs.count == 1;
  by_half_dtype(q.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (!only_few) {
      a.fewest = only_many ? 1 : kFew + 1;
      a.most = 0x7fffffff;
      const long long items = all_rows / tb200::kKvRowsOfCta + std::min<long long>(a.seqs.count, ceil_div(all_rows, a.fewest));
      if (a.cache.D <= 64) launch_rows<T, 64>(a, items, dev, stream);
      else launch_rows<T, 128>(a, items, dev, stream);
    }
    if (!only_many) {
      a.fewest = 1;
      a.most = only_few ? 0x7fffffff : kFew;
      a.row_tiles = static_cast<int>(ceil_div(a.seqs.starts == nullptr ? a.group : std::min<long long>(all_rows, kFew), tb200::kKvTokenRows));
      const long long pairs = static_cast<long long>(a.seqs.count) * a.cache.heads * a.row_tiles;
      int splits = 1;
      while (splits < 8 && pairs * splits < st.num_sms) splits *= 2;
      if (a.cache.D <= 64) launch_tokens<T, 64>(a, splits, dev, stream);
      else launch_tokens<T, 128>(a, splits, dev, stream);
    }
  });
}

}  // namespace

// ==================================================================== exported C ABI
extern "C" {

TraceaStatus tracea_kv_attention(TraceaTensorView q, TraceaKvCache cache, TraceaSequences sequences, TraceaTensorView* out,
                                 TraceaKvAttentionParams params) {
  return guarded("tracea_kv_attention", [&] { kv_attention_checked(q, cache, sequences, out, params); });
}

}  // extern "C"
