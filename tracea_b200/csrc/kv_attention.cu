// Host side of attention over the cache of keys and values: tracea_kv_attention. The reference has no counterpart.
#include "kv_host.cuh"
#include "kv_rows_sm100.cuh"
#include "kv_tokens_sm100.cuh"

namespace {

using namespace tb200_host;

template <typename Kernel>
void allow_smem(Kernel kern, std::atomic<bool> (&done)[kMaxDevices], int dev, int bytes) {
  if (done[dev].load(std::memory_order_relaxed)) return;
  TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done[dev].store(true, std::memory_order_relaxed);
}

template <typename T, int kRows, int kD, bool kExact>
void launch_tokens(tb200::KvTokensArgs& c, DeviceState& st, int dev, cudaStream_t stream) {
  constexpr int kSmem = tb200::kv_token_smem_bytes(kRows, kD);
  static std::atomic<bool> done[2][kMaxDevices];
  const tb200::KvAttentionArgs& a = c.a;
  const long long heads = static_cast<long long>(a.cache.heads) * a.row_tiles, pairs = heads * a.seqs.count;
  const int slots = tb200::kv_token_ctas(kRows) * st.num_sms;
  // The tokens that a sequence may have, as far as the host knows.
  long long most = static_cast<long long>(a.seqs.table_width) << a.cache.page_shift;
  if (a.window > 0) most = std::min<long long>(most, a.window + 16LL * tb200::kKvTokenTiles);
  // A cluster of up to eight CTAs to a sequence and head, more of them while they fill no more than the machine or have more than 2048
  // tokens each; or one line of all steps, which costs a second launch and looks at all lengths first, 6 us in all, but splits a lone long
  // sequence over every SM. us, cluster / line, for sequences x tokens (8 heads of keys, 32 of q, 128 columns): 1 x 300 5.6 / 12.4,
  // 1 x 4000 9.3 / 13.4, 1 x 16000 20.7 / 17.5, 16 x 1000 10.7 / 17.4, 16 x 4000 27 / 33, 64 x 1000 27 / 35, 64 x 0..8191 90 / 95,
  // 2 x 131000 208 / 84. All with tables that just fit: the lengths are on the device, and a table for 131072 tokens, as a captured step may
  // want, takes the line for all of them (1 x 300 12.6, 64 x 1000 35), one for 16384 splits 64 x 1000 over clusters of eight (64).
  int splits = 1;
  while (splits < 8 && splits * 16LL * tb200::kKvTokenWarps < most && (pairs * splits * 2 <= slots || most > 2048LL * splits)) splits *= 2;
  const bool shared = most <= (2 * pairs * splits >= slots ? 2048LL : 1024LL) * splits && heads <= 65535;
  if (shared) {
    auto kern = tb200::kv_tokens_kernel<T, kRows, kD, kExact, tb200::kShared>;
    allow_smem(kern, done[0], dev, kSmem);
    c.splits = splits;
    launch(kern, dim3(grid_of(static_cast<long long>(a.seqs.count) * splits), static_cast<unsigned>(heads)), tb200::kKvTokenThreads, kSmem, splits,
           kLaunchKvTokens, stream, c);
    return;
  }
  auto kern = tb200::kv_tokens_kernel<T, kRows, kD, kExact, tb200::kFlat>;
  allow_smem(kern, done[1], dev, kSmem);
  c.ctas = slots;
  const size_t rows = 2 * static_cast<size_t>(slots) * kRows;
  Scratch scratch;
  scratch.alloc(st, rows * (kD * sizeof(float) + sizeof(float2)) + slots * sizeof(int4), stream);
  c.sums = static_cast<float*>(scratch.ptr);
  c.tops = reinterpret_cast<float2*>(c.sums + rows * kD);
  c.cuts = reinterpret_cast<int4*>(c.tops + rows);
  launch(kern, static_cast<unsigned>(slots), tb200::kKvTokenThreads, kSmem, 1, kLaunchKvTokens, stream, c);
  const int join_rows = a.seqs.starts == nullptr ? std::min(a.group, kRows) : kRows;
  launch(tb200::kv_join_kernel<T, kD>, dim3(static_cast<unsigned>(slots), static_cast<unsigned>(join_rows)), 32 * tb200::kKvJoinWarps, 0, 1, kLaunchKvTokens, stream, c);
}

template <typename T, int kD>
void launch_rows(const tb200::KvAttentionArgs& a, long long items, DeviceState& st, int dev, cudaStream_t stream) {
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
  tb200::KvRowsArgs c;
  memset(&c, 0, sizeof(c));
  c.a = a;
  // Few blocks of rows leave SMs idle: their tokens are split, as long as a part has four steps where the sequences are as long as they
  // may be. us, one part / split, 32 heads to 8 of 128 columns: 256 tokens behind 8000 144 / 56, 256 behind 2000 48 / 33, 128 behind
  // 30000 496 / 86; 8 heads to 2, 500 behind 4000 82 / 34. With a table that just fits; a wider one splits short prompts as well (500 tokens
  // 18.7 -> 30.1).
  long long most = static_cast<long long>(a.seqs.table_width) << a.cache.page_shift;
  if (a.window > 0) most = std::min<long long>(most, a.window + static_cast<long long>(tb200::kKvRowsOfCta));
  const long long blocks = items * a.cache.heads;
  c.splits = static_cast<int>(std::max(1LL, std::min({st.num_sms / blocks, most / (4 * tb200::kKvRowsTokens), 16LL})));
  Scratch scratch;
  if (c.splits > 1) {
    const size_t rows = static_cast<size_t>(c.splits) * a.seqs.rows * a.cache.heads * a.group;
    scratch.alloc(st, rows * (kD * sizeof(float) + sizeof(float2)), stream);
    c.sums = static_cast<float*>(scratch.ptr);
    c.tops = reinterpret_cast<float2*>(c.sums + rows * kD);
  }
  launch(kern, grid_of(blocks * c.splits), tb200::kKvRowsThreads, kSmem, 1, kLaunchKvRows, stream, c);
  if (c.splits > 1)
    launch(tb200::kv_rows_join_kernel<T, kD>, dim3(grid_of(blocks), 8), 32 * tb200::kKvRowsJoinWarps, 0, 1, kLaunchKvRows, stream, c);
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
  if (a.cache.pages == 0) a.cache.k = a.cache.v = reinterpret_cast<uint8_t*>(q.ptr);   // what copies of no bytes point to
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
      // blocks of rows: a sequence's last one may be short
      const long long items = std::min(ceil_div(all_rows, tb200::kKvRowsOfCta) + a.seqs.count - 1,
                                       all_rows / tb200::kKvRowsOfCta + ceil_div(all_rows, a.fewest));
      if (a.cache.D <= 64) launch_rows<T, 64>(a, items, st, dev, stream);
      else launch_rows<T, 128>(a, items, st, dev, stream);
    }
    if (!only_many) {
      a.fewest = 1;
      a.most = only_few ? 0x7fffffff : kFew;
      const long long most_rows = a.seqs.starts == nullptr ? a.group : std::min<long long>(all_rows, kFew);
      a.tile_rows = most_rows <= 8 ? 8 : tb200::kKvTokenRows;
      a.row_tiles = static_cast<int>(ceil_div(most_rows, a.tile_rows));
      tb200::KvTokensArgs c;
      memset(&c, 0, sizeof(c));
      c.a = a;
      auto go = [&](auto rows) {
        constexpr int kRows = decltype(rows)::value;
        if (a.cache.D == 64) launch_tokens<T, kRows, 64, true>(c, st, dev, stream);
        else if (a.cache.D < 64) launch_tokens<T, kRows, 64, false>(c, st, dev, stream);
        else if (a.cache.D == 128) launch_tokens<T, kRows, 128, true>(c, st, dev, stream);
        else launch_tokens<T, kRows, 128, false>(c, st, dev, stream);
      };
      if (a.tile_rows == 8) go(std::integral_constant<int, 8>{});
      else go(std::integral_constant<int, tb200::kKvTokenRows>{});
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
