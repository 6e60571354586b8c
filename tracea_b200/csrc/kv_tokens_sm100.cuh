// Attention over the cache for few rows a sequence: single tokens as answers are generated, or a few drafted ones.
//
//   out = softmax(scale q K^T) V,   K = 2^ek k^, V = 2^ev v^ with a power of two per page and head, k^ and v^ in e4m3
//
// Bound by reading the cache once. The heads of q that share a head of keys (times the tokens of the sequence) are columns of the
// matrix instructions, 8 or 16 of them, and the cache's tokens (for the scores) and columns (for the results) their rows, so that few
// heads take few instructions and the cache is read once for all of them; elements of e4m3 are halves exactly, and so are those of q,
// times a power of two per row, to 11 bits of the row's largest. A warp takes 16 tokens at a time and keeps its own copies under way,
// 512 consecutive bytes each: copies by the lanes of what each multiplies, 64 bytes of eight rows, stop at 4.9 TB/s where these reach
// 6.7. In shared memory the 16-byte columns of a row are exchanged so that no two lanes meet on a bank (see below). Several CTAs of four
// warps share an SM, so that one's first loads, each of which waits for the one in front of it -- the lengths, the places of the pages,
// the pages -- and its sums' meeting lie beside the others' work. 64 sequences of 0 - 8191 tokens, 32 heads to 8 of 128: 92 - 96 us, 5.2 TB/s;
// 2 of 105000: 85 - 87 us, of which 14 are the line's set-up (below), its join and the launch of that.
//
// The work is split along the cache in one of two ways:
//   kShared    the CTAs of a cluster share a sequence and head and add up their sums through shared memory: one launch, for few tokens
//   kFlat      all sequences' and heads' steps lie in one line, of which every CTA takes an equal piece, whatever the lengths; sums of
//              what is cut go through memory and are joined by a second kernel
// The order of all sums depends on the sizes and lengths alone.
#pragma once
#include "kv_attention_sm100.cuh"

namespace tb200 {

constexpr int kKvTokenWarps = 4;
constexpr int kKvTokenThreads = 32 * kKvTokenWarps;
constexpr int kKvTokenRows = 16;               // of a tile, or 8
constexpr int kKvTokenTiles = 4;               // sequences of up to 64 rows a head of keys come here
constexpr int kKvMetaPages = 256;              // pages whose places and scales are in shared memory at a time
constexpr int kKvFlatSteps = 8;                // a CTA's piece of the line is no shorter than two steps a warp
constexpr int kKvFlatCost = 12;                // steps that take as long as a piece's beginning and end

struct KvTokensArgs {
  KvAttentionArgs a;
  int splits;                    // kShared: CTAs of a cluster
  int ctas;                      // kFlat
  float* sums;                   // kFlat: two slots a CTA of [kRows][kD] unscaled results,
  float2* tops;                  // and [kRows] of {maximum, denominator};
  int4* cuts;                    // of each CTA, the pair that begins in it and ends in another: {sequence or -1, pair, slot, last CTA}
};

// kRows: rows of a tile, 8 or 16. kD: D rounded up to 64 or 128; columns past D are zeros that nothing is read for.
// CTAs of an SM, and steps of 16 tokens that a warp has under way, one of them in work.
__host__ __device__ constexpr int kv_token_ctas(int rows) { return rows == 8 ? 4 : 3; }
__host__ __device__ constexpr int kv_token_stages(int rows) { return rows == 8 ? 3 : 4; }
__host__ __device__ constexpr int kv_token_step_bytes(int d) { return 16 * d * 2; }
__host__ __device__ constexpr int kv_token_smem_bytes(int rows, int d) {
  return kKvTokenWarps * kv_token_stages(rows) * kv_token_step_bytes(d) + kKvMetaPages * 8;
}

// What a sequence's rows see of it, in steps of 16 tokens; at least one step, so that rows that see nothing are written too.
struct TokenSpan {
  int row0, rows, length;        // rows: tokens of the call times the heads of q to a head of keys
  int see_lo, see_hi;            // tokens
  int step_lo, steps, tiles;
};
__device__ __forceinline__ TokenSpan token_span(const KvAttentionArgs& a, int seq) {
  TokenSpan s;
  int n = 1;
  s.row0 = seq;
  if (a.seqs.starts != nullptr) {
    s.row0 = max(0, min(a.seqs.starts[seq], a.seqs.rows));
    n = max(0, min(a.seqs.starts[seq + 1], a.seqs.rows) - s.row0);
  }
  s.length = max(0, min(a.seqs.lengths[seq], kMaxTokens));
  s.rows = n * a.group;
  if (s.rows < a.fewest || s.rows > a.most) s.rows = 0;
  const int begin = s.length - n;
  s.see_lo = a.window > 0 ? max(0, begin - a.window + 1) : 0;
  s.see_hi = min(s.length, a.seqs.table_width << a.cache.page_shift);
  s.step_lo = s.see_lo >> 4;
  s.steps = max(1, ((s.see_hi + 15) >> 4) - s.step_lo);
  s.tiles = (s.rows + a.tile_rows - 1) / a.tile_rows;
  return s;
}
// kFlat's line: the sequences' steps, for each in turn those of every head and tile (a pair), each pair with `cost` places in front for
// what a piece of any length takes. By a whole warp.
__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void token_totals(const KvAttentionArgs& a, long long& steps, long long& pairs) {
  steps = pairs = 0;
  for (int i = threadIdx.x & 31; i < a.seqs.count; i += 32) {
    const TokenSpan s = token_span(a, i);
    const long long n = static_cast<long long>(s.tiles) * a.cache.heads;
    pairs += n;
    steps += n * s.steps;
  }
  steps = warp_sum(steps);
  pairs = warp_sum(pairs);
}
// The sequence that place `at` of the line falls into, and where its own places begin.
__device__ __forceinline__ int token_sequence(const KvAttentionArgs& a, long long at, int cost, long long& begin) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int base = 0; base < a.seqs.count; base += 32) {
    long long mine = 0;
    if (base + lane < a.seqs.count) {
      const TokenSpan s = token_span(a, base + lane);
      mine = static_cast<long long>(s.tiles) * a.cache.heads * (s.steps + cost);
    }
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + sum > at);
    if (past != 0u) {
      const int i = __ffs(static_cast<int>(past)) - 1;
      begin = before + __shfl_sync(0xffffffffu, sum - mine, i);
      return base + i;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return -1;
}

enum { kShared = 0, kFlat = 1 };

// kExact: D == kD.
template <typename T, int kRows, int kD, bool kExact, int kSplit>
__global__ void __launch_bounds__(kKvTokenThreads, kv_token_ctas(kRows)) kv_tokens_kernel(const __grid_constant__ KvTokensArgs call) {
  using namespace ptx;
  constexpr int kSegments = kD / 64;             // of 64 columns: 16 a lane of a quad
  constexpr int kValueBytes = kD / 8;            // of a token that a lane takes
  constexpr int kTilesV = kD / 16;               // 16-column tiles of the result
  constexpr int kN = kRows / 8;                  // 8-row tiles of q
  constexpr int kStages = kv_token_stages(kRows);
  constexpr int kStep = kv_token_step_bytes(kD);
  const KvAttentionArgs& args = call.a;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_factor[kKvTokenWarps][kRows], row_m[kKvTokenWarps][kRows], row_l[kKvTokenWarps][kRows];
  __shared__ float cta_m[kRows], cta_l[kRows];
  int* const meta_page = reinterpret_cast<int*>(smem + kKvTokenWarps * kStages * kStep);
  uint32_t* const meta_scale = reinterpret_cast<uint32_t*>(meta_page + kKvMetaPages);
  griddep_launch_dependents();
  griddep_wait();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int D = kExact ? kD : args.cache.D, shift = args.cache.page_shift, page_steps = shift - 4;     // log2 of a page's steps
  const uint32_t ring = smem_u32(smem) + warp * (kStages * kStep);
  const long long page_bytes = (static_cast<long long>(args.cache.heads) << shift) * D;
  const uint32_t splits = kSplit == kShared ? cluster_ctas() : 1u, rank = kSplit == kShared ? cluster_ctarank() : 0u;

  // Rows lie 128 bytes apart, or two of 64 bytes in 128, 16-byte column c of a row (of a pair of rows) in the place of c ^ f: keys are
  // read as columns t (+ 4) of rows g, values as columns g of rows 2t (+ 1), eight lanes at a time.
  //   128-byte rows: f(r) = 2 (r / 2 % 4) ^ 4 (r % 2)        pairs of 64-byte rows p: f(p) = 2 (p % 4)
  constexpr int kCopies = kD / 32;               // of 512 bytes a step, of keys and of values each
  uint32_t copy_to[kCopies];
  int copy_row[kCopies];                         // of the step; 16: nothing to copy
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int chunk = 32 * j + lane, columns = D / 16, r = chunk / columns, c = chunk % columns;
    copy_row[j] = kExact || chunk < D ? r : 16;
    copy_to[j] = kD == 128 ? r * 128 + ((c ^ (2 * ((r >> 1) & 3)) ^ (4 * (r & 1))) * 16) : (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (2 * ((r >> 1) & 3))) * 16);
  }
  const uint32_t k_at = kD == 128 ? g * 128 + ((t ^ (2 * ((g >> 1) & 3)) ^ (4 * (g & 1))) * 16) : (g >> 1) * 128 + ((((g & 1) * 4 + t) ^ (2 * ((g >> 1) & 3))) * 16);
  const uint32_t v_at = 16 * kD + (kD == 128 ? 2 * t * 128 + ((g ^ (2 * t)) * 16) : t * 128 + (((g >> 1) ^ (2 * t)) * 16) + 8 * (g & 1));

  long long from = 0, to = 1, before = 0;        // kFlat: this CTA's piece of the line, and where its sequence begins
  long long piece0 = 0, quota = 1;
  int seq = static_cast<int>(blockIdx.x / splits);
  constexpr int cost = kKvFlatCost;
  bool used = false;                             // shared memory is, by a pair in front
  if constexpr (kSplit == kFlat) {
    long long steps, pairs;
    token_totals(args, steps, pairs);
    quota = max((steps + pairs * cost + call.ctas - 1) / call.ctas, static_cast<long long>(cost + kKvFlatSteps));
    piece0 = from = quota * blockIdx.x;
    to = min(steps + pairs * cost, from + quota);
    if (threadIdx.x == 0) call.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (from < to) seq = token_sequence(args, from, cost, before);
  }

  while (from < to) {
    const TokenSpan span = token_span(args, seq);
    int head, tile, my_lo, my_hi;                // of the sequence's steps
    long long next = to;
    if constexpr (kSplit == kFlat) {
      const int places = span.steps + cost;
      const long long all = static_cast<long long>(places) * span.tiles * args.cache.heads;
      if (from - before >= all) {                // the next sequence's turn
        before += all;
        ++seq;
        continue;
      }
      const int pair = static_cast<int>((from - before) / places);
      const long long pair0 = before + static_cast<long long>(pair) * places;
      head = pair / span.tiles;
      tile = pair % span.tiles;
      next = min(to, pair0 + places);
      my_lo = max(0, static_cast<int>(from - pair0) - cost);
      my_hi = max(0, static_cast<int>(next - pair0) - cost);
      if (my_lo == my_hi) {                      // its steps are all another CTA's
        from = next;
        continue;
      }
      if (threadIdx.x == 0 && my_lo == 0 && my_hi < span.steps)
        call.cuts[blockIdx.x] = make_int4(seq, pair, from == piece0 ? 0 : 1, static_cast<int>((pair0 + places - 1) / quota));
    } else {
      head = static_cast<int>(blockIdx.y) / args.row_tiles;
      tile = static_cast<int>(blockIdx.y) % args.row_tiles;
      if (tile >= span.tiles) return;            // the whole cluster
      my_lo = static_cast<int>(static_cast<long long>(span.steps) * rank / splits);
      my_hi = static_cast<int>(static_cast<long long>(span.steps) * (rank + 1) / splits);
    }
    const bool whole = my_lo == 0 && my_hi == span.steps;
    const int first_row = tile * kRows, rows = min(kRows, span.rows - first_row);
    const int begin = span.length - span.rows / args.group;        // position of the sequence's first row
    const int pos_lo = begin + first_row / args.group, pos_hi = begin + (first_row + rows - 1) / args.group;
    const int see_lo = span.see_lo, see_hi = span.see_hi;
    const int lo = span.step_lo + my_lo, hi = span.step_lo + my_hi;
    const uint8_t* const k_head = args.cache.k + (static_cast<long long>(head) << shift) * D;
    const uint8_t* const v_head = args.cache.v + (static_cast<long long>(head) << shift) * D;

    // Of each 8 rows of q this lane has row g as an operand, and rows 2t and 2t + 1 of scores, weights and results.
    float factor[kN][2];
    int pos[kN][2];
    uint32_t qb[kN][kSegments][4][2];
    float m[kN][2], l[kN][2], o[kN][kTilesV][4];
    bool far = false;                            // a maximum of the warp's rows is (kFar)
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int j = 0; j < kTilesV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][j][i] = 0.0f;
    }

    for (int part = lo; part < hi;) {
      // the places of this part's pages, then, while the first copies are under way, their scales
      const int page0 = part >> page_steps;
      const int part_end = min(hi, (page0 + kKvMetaPages) << page_steps);
      const int pages = ((part_end - 1) >> page_steps) - page0 + 1;
      if (part != lo || used) __syncthreads();
      if (!kExact && part == lo) {               // the columns past D, which no copy writes
        for (int i = threadIdx.x; i < kKvTokenWarps * kStages * kStep / 16; i += kKvTokenThreads)
          st_shared_v4(smem_u32(smem) + 16 * i, make_uint4(0u, 0u, 0u, 0u));
      }
      for (int i = threadIdx.x; i < pages; i += kKvTokenThreads) {
        int id = -1;
        if (page0 + i < args.seqs.table_width) id = args.seqs.table[seq * args.seqs.table_stride + page0 + i];
        meta_page[i] = id >= 0 && id < args.cache.pages ? id : -1;
      }
      __syncthreads();

      auto fetch = [&](int step, int stage) {
        const int page = meta_page[(step >> page_steps) - page0];
        const int token = (step & ((1 << page_steps) - 1)) << 4, at = step << 4;
        const long long place = page * page_bytes + token * D + 16 * lane;
        const uint8_t* const kp = k_head + place;
        const uint8_t* const vp = v_head + place;
        const uint32_t dst = ring + stage * kStep;
        if (kExact && page >= 0 && at >= see_lo && at + 16 <= see_hi) {
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            cp_async_16(dst + copy_to[j], kp + 512 * j);
            cp_async_16(dst + 16 * kD + copy_to[j], vp + 512 * j);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            if (kExact || copy_row[j] < 16) {    // tokens that no row sees become zeros: a weight of 0 takes none of them in
              const int r = at + copy_row[j];
              const bool live = page >= 0 && r >= see_lo && r < see_hi;
              cp_async_or_zero<16>(dst + copy_to[j], live ? kp + 512 * j : args.cache.k, live);
              cp_async_or_zero<16>(dst + 16 * kD + copy_to[j], live ? vp + 512 * j : args.cache.v, live);
            }
          }
        }
      };
      const int first = part + warp;
#pragma unroll
      for (int s = 0; s < kStages - 1; ++s) {
        if (first + s * kKvTokenWarps < part_end) fetch(first + s * kKvTokenWarps, s);
        cp_async_commit();
      }
      for (int i = threadIdx.x; i < pages; i += kKvTokenThreads) {
        const int id = meta_page[i];
        const long long block = static_cast<long long>(max(id, 0)) * args.cache.heads + head;
        meta_scale[i] = id >= 0 ? args.cache.k_scales[block] | (static_cast<uint32_t>(args.cache.v_scales[block]) << 8) : 0x7f7fu;
      }
      if (part == lo) {
        // q as the second operand, the columns that the first operand's lane has (see below)
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const int all = first_row + 8 * n + g;
          const bool live = 8 * n + g < rows;
          const T* p = static_cast<const T*>(args.q) + (span.row0 + (live ? all / args.group : 0)) * args.q_token +
                       (head * args.group + (live ? all % args.group : 0)) * args.q_head;
          float v[kSegments][16];
          float peak = 0.0f;
#pragma unroll
          for (int i = 0; i < kSegments; ++i) {
            const int d = 64 * i + 16 * t;
#pragma unroll
            for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
            if (live && d < D) {
              if (args.q_vec) {
                load8(p + d, reinterpret_cast<float(&)[8]>(v[i][0]));
                load8(p + d + 8, reinterpret_cast<float(&)[8]>(v[i][8]));
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[i][j] = static_cast<float>(p[d + j]);
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) peak = fmaxf(peak, fabsf(v[i][j]));
          }
          peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
          peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
          float back;
          const float up = args.sign * row_scale(peak, back);
          back *= args.scale_log2;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            factor[n][j] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + j));
            pos[n][j] = begin + (first_row + 8 * n + 2 * t + j) / args.group;
          }
#pragma unroll
          for (int i = 0; i < kSegments; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              qb[n][i][s][0] = pack_halves(v[i][4 * s] * up, v[i][4 * s + 1] * up);
              qb[n][i][s][1] = pack_halves(v[i][4 * s + 2] * up, v[i][4 * s + 3] * up);
            }
        }
      }
      __syncthreads();

      int stage = 0;
      for (int step = first; step < part_end; step += kKvTokenWarps) {
        {
          __syncwarp();                          // every lane has read what is overwritten
          const int ahead = step + (kStages - 1) * kKvTokenWarps;
          if (ahead < part_end) fetch(ahead, (stage + kStages - 1) % kStages);
          cp_async_commit();
        }
        cp_async_wait<kStages - 1>();
        __syncwarp();                            // every lane's copies are there
        const int at_page = (step >> page_steps) - page0;
        const uint32_t scales = meta_scale[at_page];
        const float k_scale = power_of_two(static_cast<int>(scales & 0xffu) - 127), ev = static_cast<float>(static_cast<int>(scales >> 8) - 127);
        const uint8_t* const src = smem + warp * (kStages * kStep) + stage * kStep;
        // scores: the order of the columns in the sums is free, so long as both operands have the same. A lane's 16 bytes of a
        // segment, of rows g and g + 8, are four instructions' worth.
        float s[kN][4];
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll
        for (int seg = 0; seg < kSegments; ++seg) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + (k_at ^ (64 * seg))), y = *reinterpret_cast<const uint4*>(src + 8 * kD + (k_at ^ (64 * seg)));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a[4];
            halves_of_e4m3(xs[j], a[0], a[2]);
            halves_of_e4m3(ys[j], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_16x8x16(s[n], a, qb[n][seg][j][0], qb[n][seg][j][1]);
          }
        }
        // s[n][2 half + j]: token g + 8 half of the step, row 8n + 2t + j
        const int at = step << 4;
        const bool page_there = meta_page[at_page] >= 0;
        if (!page_there || at + 16 > see_hi || (args.causal && at + 15 > pos_lo) || (args.window > 0 && at <= pos_hi - args.window)) {
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int token = at + g + 8 * (i >> 1), p = pos[n][i & 1];
              const bool seen = page_there && token < see_hi && (!args.causal || token <= p) && (args.window == 0 || token > p - args.window);
              s[n][i] = seen ? s[n][i] * (factor[n][i & 1] * k_scale) + ev : -INFINITY;
            }
        } else {
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = s[n][i] * (factor[n][i & 1] * k_scale) + ev;
        }
        bool grown = far;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) grown = grown || fmaxf(s[n][j], s[n][2 + j]) > m[n][j] + kSlack;
        if (__any_sync(0xffffffffu, grown)) {
          bool mine = false;
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float p = fmaxf(fmaxf(s[n][j], s[n][2 + j]), m[n][j]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, x));
              const float shrink = p == m[n][j] ? 1.0f : exp2_ftz(m[n][j] - p);
              m[n][j] = p;
              mine = mine || is_far(p);
              l[n][j] *= shrink;
#pragma unroll
              for (int v = 0; v < kTilesV; ++v) {
                o[n][v][j] *= shrink;
                o[n][v][2 + j] *= shrink;
              }
            }
          far = __any_sync(0xffffffffu, mine);
        }
        if (far) {
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = m[n][i & 1] == -INFINITY ? s[n][i] : s[n][i] - m[n][i & 1] + kLift;
        }
        const float unscale = power_of_two(127 - static_cast<int>(scales >> 8));
        uint32_t pb[kN][2];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float base = m[n][j] == -INFINITY || far ? 0.0f : m[n][j] - kLift;      // 0: a row that has seen nothing, or see above
            s[n][j] = exp2_ftz(s[n][j] - base);
            s[n][2 + j] = exp2_ftz(s[n][2 + j] - base);
            l[n][j] += (s[n][j] + s[n][2 + j]) * unscale;
          }
          // from two rows of a token to two tokens of a row
          pb[n][0] = transposed_8x8(pack_halves(s[n][0], s[n][1]));
          pb[n][1] = transposed_8x8(pack_halves(s[n][2], s[n][3]));
        }
        // values: two tokens' elements of a column make a word of the first operand
        uint32_t w[4][kValueBytes / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kValueBytes == 16) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + (i >> 1) * 1024 + (i & 1) * 128 + (v_at ^ (64 * (i & 1))));
            w[i][0] = x.x;
            w[i][1] = x.y;
            w[i][2] = x.z;
            w[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src + (i >> 1) * 512 + (v_at ^ (64 * (i & 1))));
            w[i][0] = x.x;
            w[i][1] = x.y;
          }
        }
#pragma unroll
        for (int q = 0; q < kValueBytes / 4; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {          // columns 4q + 2h and the next of the lane's
            const uint32_t mix = h == 0 ? 0x5140 : 0x7362;
            uint32_t a[4];
            halves_of_e4m3(__byte_perm(w[0][q], w[1][q], mix), a[0], a[1]);
            halves_of_e4m3(__byte_perm(w[2][q], w[3][q], mix), a[2], a[3]);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_16x8x16(o[n][2 * q + h], a, pb[n][0], pb[n][1]);
          }
        stage = (stage + 1) % kStages;
      }
      cp_async_wait_all();
      part = part_end;
    }

    // The sums of the warps, always in the same order. o[n][v][2i + j]: row 8n + 2t + j, column kValueBytes g + 2v + i.
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
        if (g == 0) {
          row_m[warp][8 * n + 2 * t + j] = m[n][j];
          row_l[warp][8 * n + 2 * t + j] = l[n][j];
        }
      }
    __syncthreads();
    constexpr int kRowFloats = kD + 4;                      // of a row of partial sums: keeps 8 rows off each other's banks
    float* const part = reinterpret_cast<float*>(smem);
    static_assert(kKvTokenWarps * kRows * kRowFloats * 4 <= kv_token_smem_bytes(kRows, kD), "the partial sums lie over the ring");
    if (threadIdx.x < kRows) {
      float top = -INFINITY, total = 0.0f;
#pragma unroll
      for (int w = 0; w < kKvTokenWarps; ++w) top = fmaxf(top, row_m[w][threadIdx.x]);
#pragma unroll
      for (int w = 0; w < kKvTokenWarps; ++w) {
        const float f = part_factor(row_m[w][threadIdx.x], row_l[w][threadIdx.x], top);
        row_factor[w][threadIdx.x] = f;
        total += f * row_l[w][threadIdx.x];
      }
      cta_m[threadIdx.x] = top;
      cta_l[threadIdx.x] = total;
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int v = 0; v < kTilesV; ++v)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float2*>(part + (warp * kRows + 8 * n + 2 * t + j) * kRowFloats + kValueBytes * g + 2 * v) =
              make_float2(o[n][v][j], o[n][v][2 + j]);
    __syncthreads();
    auto sum_of_warps = [&](int r, int d) {
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kKvTokenWarps; ++w) add_scaled(sum, *reinterpret_cast<const float4*>(part + (w * kRows + r) * kRowFloats + d), row_factor[w][r]);
      return sum;
    };
    auto write = [&](int r, int d, const float4& sum, float total) {
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      const int all = first_row + r;
      T* p = static_cast<T*>(args.out) + (span.row0 + all / args.group) * args.out_token + (head * args.group + all % args.group) * args.out_head + d;
      store_4(p, sum, inv, args.out_vec);
    };
    const int items = rows * (kD / 4);                      // of four columns
    if (kSplit == kFlat || splits == 1) {
      const int slot = 2 * static_cast<int>(blockIdx.x) + (from == piece0 ? 0 : 1);
      for (int i = threadIdx.x; i < items; i += kKvTokenThreads) {
        const int r = i / (kD / 4), d = 4 * (i % (kD / 4));
        if (d >= D) continue;
        const float4 sum = sum_of_warps(r, d);
        if (whole) write(r, d, sum, cta_l[r]);
        else *reinterpret_cast<float4*>(call.sums + (static_cast<long long>(slot) * kRows + r) * kD + d) = sum;
      }
      if (!whole && static_cast<int>(threadIdx.x) < rows)
        call.tops[static_cast<long long>(slot) * kRows + threadIdx.x] = make_float2(cta_m[threadIdx.x], cta_l[threadIdx.x]);
    } else {
      for (int i = threadIdx.x; i < items; i += kKvTokenThreads) {
        const int r = i / (kD / 4), d = 4 * (i % (kD / 4));
        const float4 sum = sum_of_warps(r, d);
        *reinterpret_cast<float4*>(part + r * kRowFloats + d) = sum;     // over warp 0's, which this thread alone reads here
      }
      cluster_sync();
      // every CTA finishes a share of the rows' columns
      const int share = (items + static_cast<int>(splits) - 1) / static_cast<int>(splits);
      for (int i = static_cast<int>(rank) * share + threadIdx.x; i < min(items, (static_cast<int>(rank) + 1) * share); i += kKvTokenThreads) {
        const int r = i / (kD / 4), d = 4 * (i % (kD / 4));
        if (d >= D) continue;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float total = 0.0f, top = -INFINITY;
        for (uint32_t c = 0; c < splits; ++c) top = fmaxf(top, ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_m[r]), c)));
        for (uint32_t c = 0; c < splits; ++c) {
          const float cm = ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_m[r]), c)), cl = ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_l[r]), c));
          const float f = part_factor(cm, cl, top);
          add_scaled(sum, ld_shared_cluster_f4(mapa_cluster(smem_u32(part + r * kRowFloats + d), c)), f);
          total += f * cl;
        }
        write(r, d, sum, total);
      }
      cluster_sync();                                       // nobody leaves while others read its sums
    }
    if constexpr (kSplit == kShared) break;
    from = next;
    used = true;
  }
}

// kFlat's second kernel: for each CTA of the first, the pair that begins in it and ends in another, a row to a CTA, its warps the pieces
// in turn.
constexpr int kKvJoinWarps = 8;
template <typename T, int kD>
__global__ void __launch_bounds__(32 * kKvJoinWarps) kv_join_kernel(const __grid_constant__ KvTokensArgs call) {
  using namespace ptx;
  const KvAttentionArgs& args = call.a;
  __shared__ float totals[kKvJoinWarps];
  __shared__ float4 sums[kKvJoinWarps][kD / 4];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = static_cast<int>(blockIdx.x), row = static_cast<int>(blockIdx.y);
  const int4 cut = call.cuts[c0];                           // {sequence, pair, slot, last CTA}
  if (cut.x < 0) return;
  const TokenSpan span = token_span(args, cut.x);
  const int head = cut.y / span.tiles, all = cut.y % span.tiles * args.tile_rows + row;
  if (all >= span.rows) return;
  auto slot = [&](int c) { return (2 * static_cast<long long>(c) + (c == c0 ? cut.z : 0)) * args.tile_rows + row; };
  float top = -INFINITY;
  for (int c = c0 + lane; c <= cut.w; c += 32) top = fmaxf(top, call.tops[slot(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float total = 0.0f;
  const bool mine = 4 * lane < args.cache.D;
#pragma unroll 4
  for (int c = c0 + warp; c <= cut.w; c += kKvJoinWarps) {
    const float2 t = call.tops[slot(c)];
    const float f = part_factor(t.x, t.y, top);
    total += f * t.y;
    if (mine) add_scaled(sum, *reinterpret_cast<const float4*>(call.sums + slot(c) * kD + 4 * lane), f);
  }
  if (4 * lane < kD) sums[warp][lane] = sum;
  if (lane == 0) totals[warp] = total;
  __syncthreads();
  if (warp != 0 || !mine) return;
  for (int w = 1; w < kKvJoinWarps; ++w) {
    add_scaled(sum, sums[w][lane], 1.0f);
    total += totals[w];
  }
  T* p = static_cast<T*>(args.out) + (span.row0 + all / args.group) * args.out_token + (head * args.group + all % args.group) * args.out_head + 4 * lane;
  store_4(p, sum, total == 0.0f ? 0.0f : 1.0f / total, args.out_vec);
}

}  // namespace tb200
