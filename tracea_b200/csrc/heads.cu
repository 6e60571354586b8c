// Host side of the operators on rows of heads: tracea_head_norm_rotate, tracea_kv_append. The reference has no counterpart.
#include "kv_host.cuh"

namespace {

using namespace tb200_host;

// f(lanes of a row, or 0: a warp, column by column; whether a rotation's pairs are neighbours).
template <typename F>
void by_head_lanes(int lanes, bool neighbours, F&& f) {
  auto with = [&](auto row_lanes) {
    if constexpr (decltype(row_lanes)::value > 0) {      // the scalar form goes by its columns alone
      if (neighbours) return f(row_lanes, std::true_type{});
    }
    f(row_lanes, std::false_type{});
  };
  switch (lanes) {
    case 1: with(std::integral_constant<int, 1>{}); break;
    case 2: with(std::integral_constant<int, 2>{}); break;
    case 4: with(std::integral_constant<int, 4>{}); break;
    case 8: with(std::integral_constant<int, 8>{}); break;
    case 16: with(std::integral_constant<int, 16>{}); break;
    default: with(std::integral_constant<int, 0>{});
  }
}

// Whether a rotation and the columns suit lanes of 16 columns (see HeadLane).
bool lanes_of_16(long long cols, const tb200::Rotation& rot) { return cols % 16 == 0 && rot.pairs % 8 == 0; }

void head_rotate_checked(const TraceaHeads* q, const TraceaHeads* k, TraceaNormKind kind, float eps, const TraceaRotation* rotation,
                         const TraceaTensorView* positions, void* stream) {
  const TraceaHeads* given[2] = {q != nullptr ? q : k, q != nullptr ? k : nullptr};
  if (given[0] == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "neither queries nor keys are given");
  const int dev = given[0]->x.device_id;
  if (dev < 0) TB_FAIL(TRACEA_INVALID_PARAMS, "tracea_head_norm_rotate takes device tensors (device_id >= 0)");
  tb200::HeadRotateArgs a;
  memset(&a, 0, sizeof(a));
  Heads first;
  bool vec = true;
  long long heads = 0;
  for (int i = 0; i < 2 && given[i] != nullptr; ++i) {
    const char* name = given[i] == q ? "q" : "k";
    if (given[i]->y == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "%s has no output", name);
    const Heads x = load_heads(given[i]->x, name, dev), y = load_heads(*given[i]->y, "the output", dev);
    if (i == 0) first = x;
    check_like(x, name, first, "q");
    check_like(y, "the output", x, name);
    if (y.heads != x.heads) TB_FAIL(TRACEA_INVALID_PARAMS, "the output has %lld heads, %s has %lld", y.heads, name, x.heads);
    check_heads_output(y, "the output");
    int f32;
    const void* w = load_head_weight(given[i]->weight, "weight", dev, x.cols, x.dtype, f32);
    a.rows[i] = load_head_rows(x, &y, w, f32);
    vec = vec && x.vec && y.vec;
    heads += x.heads;
  }
  if (first.cols > tb200::kHeadMaxColumns || first.cols % 2 != 0)
    TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "heads of %lld columns: an even number up to %d", first.cols, tb200::kHeadMaxColumns);
  a.norm = load_head_norm(kind, eps);
  a.eps = eps;
  a.rot = load_rotation(rotation, first.cols);
  if (a.rot.pairs > 0) {
    if (positions == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "a rotation takes positions");
    check_int_vector(*positions, "positions", dev, first.tokens);
    a.positions = static_cast<const int*>(positions->ptr);
  }
  if (first.tokens == 0) return;
  a.tokens = static_cast<int>(first.tokens);
  a.D = static_cast<int>(first.cols);
  vec = vec && lanes_of_16(first.cols, a.rot);
  const int lanes = vec ? head_lanes(first.cols) : 32;
  const long long passes = ceil_div(a.rows[0].heads, 32 / lanes) + ceil_div(a.rows[1].heads, 32 / lanes);
  if (passes > 0xffff) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%lld heads", heads);
  a.passes = static_cast<int>(passes);
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  // Warps that share a token compute its angles each for itself, so no more of them than give the machine its 32 an SM.
  const long long wanted = ceil_div(32LL * st.num_sms, first.tokens);
  const dim3 grid(grid_of(ceil_div(first.tokens, tb200::kHeadThreads / 32)), static_cast<unsigned>(std::max(1LL, std::min(passes, wanted))));
  by_dtype(first.dtype, [&](auto tag) {
    by_head_lanes(vec ? lanes : 0, a.rot.interleaved != 0, [&](auto row_lanes, auto neighbours) {
      launch(tb200::head_rotate_kernel<decltype(tag), decltype(row_lanes)::value, decltype(neighbours)::value>, grid, tb200::kHeadThreads, 0, 1,
             kLaunchHeads, static_cast<cudaStream_t>(stream), a);
    });
  });
}

template <typename T, int kLanes, bool kNeighbours, int kRows>
void launch_append(const tb200::KvAppendArgs& a, dim3 grid, int dev, cudaStream_t stream) {
  const int smem = a.turn_rows * a.rot.pairs * static_cast<int>(sizeof(float2));
  auto kern = tb200::kv_append_kernel<T, kLanes, kNeighbours, kRows>;
  constexpr int kMost = tb200::kCacheMaxPage * (tb200::kCacheMaxColumns / 2) * static_cast<int>(sizeof(float2));
  static std::atomic<bool> done[kMaxDevices];
  if (smem > 40 * 1024 && !done[dev].load(std::memory_order_relaxed)) {
    TB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    done[dev].store(true, std::memory_order_relaxed);
  }
  launch(kern, grid, tb200::kHeadThreads, smem, 1, kLaunchHeads, stream, a);
}

void kv_append_checked(const TraceaKvCache& cache, const TraceaSequences& seqs, const TraceaTensorView& kv, const TraceaTensorView& vv,
                       const TraceaTensorView* k_weight, const TraceaHeads* q, TraceaNormKind kind, float eps,
                       const TraceaRotation* rotation, void* stream) {
  tb200::KvAppendArgs a;
  memset(&a, 0, sizeof(a));
  a.cache = load_cache(cache);
  const int dev = cache.device_id;
  const Heads k = load_heads(kv, "k", dev), v = load_heads(vv, "v", dev);
  check_like(v, "v", k, "k");
  if (k.heads != a.cache.heads || v.heads != a.cache.heads || k.cols != a.cache.D)
    TB_FAIL(TRACEA_INVALID_PARAMS, "k has %lld heads of %lld columns, v %lld, the cache %d of %d", k.heads, k.cols, v.heads, a.cache.heads, a.cache.D);
  a.seqs = load_sequences(seqs, dev, k.tokens);
  int f32;
  const void* w = load_head_weight(k_weight, "k_weight", dev, k.cols, k.dtype, f32);
  a.k = load_head_rows(k, nullptr, w, f32);
  a.v = v.ptr;
  a.v_token = v.token_stride;
  a.v_head = v.head_stride;
  bool vec = k.vec && v.vec;
  if (q != nullptr) {
    if (q->y == nullptr) TB_FAIL(TRACEA_INVALID_PARAMS, "q has no output");
    const Heads x = load_heads(q->x, "q", dev), y = load_heads(*q->y, "the output", dev);
    check_like(x, "q", k, "k");
    check_like(y, "the output", x, "q");
    if (y.heads != x.heads) TB_FAIL(TRACEA_INVALID_PARAMS, "the output has %lld heads, q has %lld", y.heads, x.heads);
    if (x.heads % k.heads != 0) TB_FAIL(TRACEA_INVALID_PARAMS, "%lld heads of q are no multiple of the %lld of k", x.heads, k.heads);
    if (x.heads > tb200::kCacheMostQueryHeads) TB_FAIL(TRACEA_UNSUPPORTED_CONFIG, "%lld heads of q: up to %lld", x.heads, tb200::kCacheMostQueryHeads);
    check_heads_output(y, "the output");
    w = load_head_weight(q->weight, "q_weight", dev, k.cols, k.dtype, f32);
    a.q = load_head_rows(x, &y, w, f32);
    a.group = static_cast<int>(x.heads / k.heads);
    vec = vec && x.vec && y.vec;
  }
  a.norm = load_head_norm(kind, eps);
  a.eps = eps;
  a.rot = load_rotation(rotation, k.cols);
  if (k.tokens == 0 || a.seqs.count == 0) return;
  vec = vec && lanes_of_16(k.cols, a.rot);
  const int lanes = vec ? head_lanes(k.cols) : 32;
  const int size = 1 << a.cache.page_shift;
  a.turn_rows = a.seqs.starts != nullptr ? size : 1;
  a.turn_lanes = 1;
  while (a.turn_lanes < a.rot.pairs) a.turn_lanes *= 2;
  DeviceGuard guard(dev);
  DeviceState& st = device_state(dev);
  // Pages that get tokens: one a sequence, and with n tokens at most ceil((n - 1) / P) more.
  const long long pages = a.seqs.starts != nullptr ? std::min(k.tokens, k.tokens / size + 2LL * a.seqs.count) : a.seqs.count;
  // All heads of a page share its angles; where the pages would leave a quarter of the machine's two CTAs an SM idle the heads are split
  // over CTAs all the same.
  a.heads_per_cta = a.cache.heads;
  while (a.heads_per_cta > 1 && pages * ceil_div(a.cache.heads, a.heads_per_cta) < 3LL * st.num_sms / 2) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const dim3 grid(grid_of(pages), static_cast<unsigned>(ceil_div(a.cache.heads, a.heads_per_cta)));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rows = a.seqs.starts == nullptr ? 1 : std::max(1, size * lanes / tb200::kHeadThreads);
  by_dtype(k.dtype, [&](auto tag) {
    by_head_lanes(vec ? lanes : 0, a.rot.interleaved != 0, [&](auto row_lanes, auto neighbours) {
      using T = decltype(tag);
      constexpr int kLanes = decltype(row_lanes)::value;
      constexpr bool kNeighbours = decltype(neighbours)::value;
      if constexpr (kLanes == 0) {
        if (rows <= 4) launch_append<T, 0, false, 4>(a, grid, dev, s);
        else launch_append<T, 0, false, 16>(a, grid, dev, s);
      } else if constexpr (kLanes <= 8) {
        if (rows <= 1) launch_append<T, kLanes, kNeighbours, 1>(a, grid, dev, s);
        else if constexpr (kLanes >= 4) {
          if (rows == 2) launch_append<T, kLanes, kNeighbours, 2>(a, grid, dev, s);
          else if constexpr (kLanes == 8) launch_append<T, kLanes, kNeighbours, 4>(a, grid, dev, s);
        }
      }
    });
  });
}

}  // namespace

// ==================================================================== exported C ABI
extern "C" {

TraceaStatus tracea_head_norm_rotate(const TraceaHeads* q, const TraceaHeads* k, TraceaNormKind kind, float eps,
                                     const TraceaRotation* rotation, const TraceaTensorView* positions, void* stream) {
  return guarded("tracea_head_norm_rotate", [&] { head_rotate_checked(q, k, kind, eps, rotation, positions, stream); });
}
TraceaStatus tracea_kv_append(TraceaKvCache cache, TraceaSequences sequences, TraceaTensorView k, TraceaTensorView v,
                              const TraceaTensorView* k_weight, const TraceaHeads* q, TraceaNormKind kind, float eps,
                              const TraceaRotation* rotation, void* stream) {
  return guarded("tracea_kv_append", [&] { kv_append_checked(cache, sequences, k, v, k_weight, q, kind, eps, rotation, stream); });
}

}  // extern "C"
