// Attention over the cache for few rows a sequence: single tokens as answers are generated, or a few drafted ones.
//
//   out = softmax(scale q K^T) V,   K = 2^ek k^, V = 2^ev v^ with a power of two per page and head, k^ and v^ in e4m3
//
// Bound by reading the cache once. The heads of q that share a head of keys (times the tokens of the sequence) are the 16 rows of the
// matrix instructions, so the cache is read once for all of them; elements of e4m3 are halves exactly, and so are those of q, times a
// power of two per row, to 11 bits of the row's largest. A cluster shares a sequence's tokens, its CTAs' warps take 16 of them in turn,
// and each warp keeps its own copies under way: a lane copies just the bytes that it will multiply, into its own places of shared
// memory, which needs no barrier and gives no bank conflicts. The warps' sums meet at the end, in a fixed order.
#pragma once
#include "kv_attention_sm100.cuh"

namespace tb200 {

constexpr int kKvTokenWarps = 8;
constexpr int kKvTokenThreads = 32 * kKvTokenWarps;
constexpr int kKvTokenStages = 6;              // steps of 16 tokens that a warp has under way
constexpr int kKvTokenRows = 16;
constexpr int kKvTokenTiles = 4;               // sequences of up to 64 rows a head of keys come here
constexpr int kKvMetaPages = 1024;             // pages whose places and scales are in shared memory at a time

// kD: D rounded up to 64 or 128; columns past D are zeros that nothing is read for.
template <int kD>
__host__ __device__ constexpr int kv_token_step_bytes() { return 16 * kD * 2; }
template <int kD>
__host__ __device__ constexpr int kv_token_smem_bytes() {
  return kKvTokenWarps * kKvTokenStages * kv_token_step_bytes<kD>() + kKvMetaPages * 8;
}

template <typename T, int kD>
__global__ void __launch_bounds__(kKvTokenThreads, 1) kv_tokens_kernel(const __grid_constant__ KvAttentionArgs args) {
  using namespace ptx;
  constexpr int kSegments = kD / 64;             // of 64 columns: 16 a lane of a quad
  constexpr int kValueBytes = kD / 8;            // of a token that a lane takes
  constexpr int kTilesV = kD / 8;                // 8-column tiles of the result
  constexpr int kStep = kv_token_step_bytes<kD>();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_factor[kKvTokenWarps][kKvTokenRows], row_m[kKvTokenWarps][kKvTokenRows], row_l[kKvTokenWarps][kKvTokenRows];
  __shared__ float cta_m[kKvTokenRows], cta_l[kKvTokenRows];
  int* const meta_page = reinterpret_cast<int*>(smem + kKvTokenWarps * kKvTokenStages * kStep);
  uint32_t* const meta_scale = reinterpret_cast<uint32_t*>(meta_page + kKvMetaPages);
  griddep_launch_dependents();
  griddep_wait();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t splits = cluster_ctas(), rank = cluster_ctarank();
  const int seq = static_cast<int>(blockIdx.x / splits);
  const int head = static_cast<int>(blockIdx.y) / args.row_tiles, tile = static_cast<int>(blockIdx.y) % args.row_tiles;
  int row0 = seq, n = 1;
  if (args.seqs.starts != nullptr) {
    row0 = max(0, min(args.seqs.starts[seq], args.seqs.rows));
    n = max(0, min(args.seqs.starts[seq + 1], args.seqs.rows) - row0);
  }
  const int length = max(0, min(args.seqs.lengths[seq], kMaxTokens));
  const long long all_rows = static_cast<long long>(n) * args.group;
  const int first_row = tile * kKvTokenRows;
  if (all_rows < args.fewest || all_rows > args.most || first_row >= all_rows) return;      // the whole cluster
  const int rows = static_cast<int>(min(static_cast<long long>(kKvTokenRows), all_rows - first_row));
  const int D = args.cache.D, shift = args.cache.page_shift;

  // what this tile's rows see of the sequence: positions of the first and the last row
  const int begin = length - n;
  const int pos_lo = begin + first_row / args.group, pos_hi = begin + (first_row + rows - 1) / args.group;
  const int see_lo = args.window > 0 ? max(0, pos_lo - args.window + 1) : 0;
  const int see_hi = min(args.causal ? max(0, pos_hi + 1) : length, args.seqs.table_width << shift);
  // this CTA's share of it, in steps of 16 tokens
  const int step_lo = see_lo >> 4, steps_all = max(0, ((see_hi + 15) >> 4) - step_lo);
  const int my_lo = step_lo + static_cast<int>(static_cast<long long>(steps_all) * rank / splits);
  const int my_hi = step_lo + static_cast<int>(static_cast<long long>(steps_all) * (rank + 1) / splits);

  // rows of q as the first operand: rows g and g + 8, the columns that the second operand's lane has (see below)
  uint32_t qa[kSegments][4][4];
  float factor[2];
  int pos[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g + 8 * half, all = first_row + r;
    const bool live = r < rows;
    pos[half] = begin + all / args.group;
    const T* p = static_cast<const T*>(args.q) + (row0 + (live ? all / args.group : 0)) * args.q_token +
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
    factor[half] = back * args.scale_log2;
#pragma unroll
    for (int i = 0; i < kSegments; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        qa[i][s][half] = pack_halves(v[i][4 * s] * up, v[i][4 * s + 1] * up);
        qa[i][s][half + 2] = pack_halves(v[i][4 * s + 2] * up, v[i][4 * s + 3] * up);
      }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  float o[kTilesV][4];
#pragma unroll
  for (int j = 0; j < kTilesV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;

  const uint32_t ring = smem_u32(smem) + warp * (kKvTokenStages * kStep);
  const long long page_bytes = (static_cast<long long>(args.cache.heads) << shift) * D;
  const uint8_t* const k_head = args.cache.k + (static_cast<long long>(head) << shift) * D;
  const uint8_t* const v_head = args.cache.v + (static_cast<long long>(head) << shift) * D;
  const int page_steps = shift - 4;              // log2 of a page's steps

  for (int part = my_lo; part < my_hi;) {
    // the places of this part's pages, then, while the first copies are under way, their scales
    const int page0 = part >> page_steps;
    const int part_end = min(my_hi, (page0 + kKvMetaPages) << page_steps);
    const int pages = ((part_end - 1) >> page_steps) - page0 + 1;
    if (part != my_lo) __syncthreads();
    for (int i = threadIdx.x; i < pages; i += kKvTokenThreads) {
      const int id = args.seqs.table[seq * args.seqs.table_stride + page0 + i];
      meta_page[i] = id >= 0 && id < args.cache.pages ? id : -1;
    }
    __syncthreads();

    // a step's copies: of key row 8i + g, 16 bytes of each segment; of value rows 8i + 2t, + 1, the lane's columns
    auto fetch = [&](int step, int stage) {
      const int page = meta_page[(step >> page_steps) - page0];
      const int token = (step & ((1 << page_steps) - 1)) << 4;
      const uint8_t* kp = k_head + page * page_bytes + static_cast<long long>(token) * D;
      const uint8_t* vp = v_head + page * page_bytes + static_cast<long long>(token) * D;
      const uint32_t dst = ring + stage * kStep;
      const int at = step << 4;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < kSegments; ++s) {
          const int r = 8 * i + g, d = 64 * s + 16 * t;
          const bool live = page >= 0 && d < D && at + r < see_hi;
          cp_async_or_zero<16>(dst + ((i * kSegments + s) * 32 + lane) * 16, live ? kp + r * D + d : args.cache.k, live);
        }
      const uint32_t vdst = dst + 16 * kD;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * (i >> 1) + 2 * t + (i & 1), d = kValueBytes * g;
        const bool live = page >= 0 && d < D && at + r < see_hi && at + r >= see_lo;
        cp_async_or_zero<kValueBytes>(vdst + (i * 32 + lane) * kValueBytes, live ? vp + r * D + d : args.cache.v, live);
      }
    };
    const int first = part + warp;
#pragma unroll
    for (int s = 0; s < kKvTokenStages - 1; ++s) {
      if (first + s * kKvTokenWarps < part_end) fetch(first + s * kKvTokenWarps, s);
      cp_async_commit();
    }
    for (int i = threadIdx.x; i < pages; i += kKvTokenThreads) {
      const int id = meta_page[i];
      const long long block = static_cast<long long>(max(id, 0)) * args.cache.heads + head;
      meta_scale[i] = id >= 0 ? args.cache.k_scales[block] | (static_cast<uint32_t>(args.cache.v_scales[block]) << 8) : 0x7f7fu;
    }
    __syncthreads();

    int stage = 0;
    for (int step = first; step < part_end; step += kKvTokenWarps) {
      {
        const int ahead = step + (kKvTokenStages - 1) * kKvTokenWarps;
        const int slot = stage == 0 ? kKvTokenStages - 1 : stage - 1;
        if (ahead < part_end) fetch(ahead, slot);
        cp_async_commit();
      }
      cp_async_wait<kKvTokenStages - 1>();
      const int at_page = (step >> page_steps) - page0;
      const uint32_t scales = meta_scale[at_page];
      const float k_scale = power_of_two(static_cast<int>(scales & 0xffu) - 127), ev = static_cast<float>(static_cast<int>(scales >> 8) - 127);
      const uint32_t src = ring + stage * kStep;
      // scores: the order of the columns in the sums is free, so long as both operands have the same. A lane's 16 bytes of a
      // segment are four instructions' worth.
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll
        for (int seg = 0; seg < kSegments; ++seg) {
          const uint4 w = ld_shared_v4(src + ((i * kSegments + seg) * 32 + lane) * 16);
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_16x8x16(s[i], qa[seg][j], halves_of_e4m3(words[j] & 0xffffu), halves_of_e4m3(words[j] >> 16));
        }
      }
      // s[i][2 half + j]: row g + 8 half, token 8i + 2t + j of the step
      const int at = step << 4;
      float peak[2] = {-INFINITY, -INFINITY};
      const float c[2] = {factor[0] * k_scale, factor[1] * k_scale};
      const bool page_there = meta_page[at_page] >= 0;
      if (!page_there || at + 16 > see_hi || (args.causal && at + 15 > pos_lo) || (args.window > 0 && at <= pos_hi - args.window)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int token = at + 8 * i + 2 * t + j;
              const bool seen = page_there && token < see_hi && (!args.causal || token <= pos[half]) &&
                                (args.window == 0 || token > pos[half] - args.window);
              s[i][2 * half + j] = seen ? s[i][2 * half + j] * c[half] + ev : -INFINITY;
            }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = s[i][j] * c[j >> 1] + ev;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
        peak[half] = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
      if (__any_sync(0xffffffffu, peak[0] > m[0] + kSlack || peak[1] > m[1] + kSlack)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float p = fmaxf(peak[half], m[half]);
          p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, 1));
          p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, 2));
          const float shrink = p == m[half] ? 1.0f : exp2_ftz(m[half] - p);
          m[half] = p;
          l[half] *= shrink;
#pragma unroll
          for (int j = 0; j < kTilesV; ++j) {
            o[j][2 * half] *= shrink;
            o[j][2 * half + 1] *= shrink;
          }
        }
      }
      const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};   // a row that has seen nothing
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = exp2_ftz(s[i][j] - base[j >> 1]);
          sum[j >> 1] += s[i][j];
        }
      const float unscale = power_of_two(127 - static_cast<int>(scales >> 8));
      l[0] += sum[0] * unscale;
      l[1] += sum[1] * unscale;
      const uint32_t pa[4] = {pack_halves(s[0][0], s[0][1]), pack_halves(s[0][2], s[0][3]), pack_halves(s[1][0], s[1][1]),
                              pack_halves(s[1][2], s[1][3])};
      // values: two tokens' elements of a column make a word of the second operand
      const uint32_t vsrc = src + 16 * kD;
      uint32_t w[4][kValueBytes / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kValueBytes == 16) {
          const uint4 x = ld_shared_v4(vsrc + (i * 32 + lane) * 16);
          w[i][0] = x.x;
          w[i][1] = x.y;
          w[i][2] = x.z;
          w[i][3] = x.w;
        } else {
          const uint2 x = ld_shared_v2(vsrc + (i * 32 + lane) * 8);
          w[i][0] = x.x;
          w[i][1] = x.y;
        }
      }
#pragma unroll
      for (int q = 0; q < kValueBytes / 4; ++q) {
        const uint32_t lo0 = __byte_perm(w[0][q], w[1][q], 0x5140), hi0 = __byte_perm(w[0][q], w[1][q], 0x7362);
        const uint32_t lo1 = __byte_perm(w[2][q], w[3][q], 0x5140), hi1 = __byte_perm(w[2][q], w[3][q], 0x7362);
        mma_16x8x16(o[4 * q], pa, halves_of_e4m3(lo0 & 0xffffu), halves_of_e4m3(lo1 & 0xffffu));
        mma_16x8x16(o[4 * q + 1], pa, halves_of_e4m3(lo0 >> 16), halves_of_e4m3(lo1 >> 16));
        mma_16x8x16(o[4 * q + 2], pa, halves_of_e4m3(hi0 & 0xffffu), halves_of_e4m3(hi1 & 0xffffu));
        mma_16x8x16(o[4 * q + 3], pa, halves_of_e4m3(hi0 >> 16), halves_of_e4m3(hi1 >> 16));
      }
      stage = stage == kKvTokenStages - 1 ? 0 : stage + 1;
    }
    cp_async_wait_all();
    part = part_end;
  }

  // The sums of the warps, then those of the cluster's CTAs, always in the same order. o[j][2 half + i]: row g + 8 half, column
  // kValueBytes (2t + i) + j.
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    if (t == 0) {
      row_m[warp][g + 8 * half] = m[half];
      row_l[warp][g + 8 * half] = l[half];
    }
  }
  __syncthreads();
  constexpr int kRowFloats = kD + 4;                      // of a row of partial sums: keeps 8 rows off each other's banks
  float* const part = reinterpret_cast<float*>(smem);
  static_assert(kKvTokenWarps * kKvTokenRows * kRowFloats * 4 <= kv_token_smem_bytes<kD>(), "the partial sums lie over the ring");
  if (threadIdx.x < kKvTokenRows) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kKvTokenWarps; ++w) top = fmaxf(top, row_m[w][threadIdx.x]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kKvTokenWarps; ++w) {
      const float f = row_m[w][threadIdx.x] == -INFINITY ? (row_l[w][threadIdx.x] != row_l[w][threadIdx.x] ? 1.0f : 0.0f) : exp2_ftz(row_m[w][threadIdx.x] - top);
      row_factor[w][threadIdx.x] = f;
      total += f * row_l[w][threadIdx.x];
    }
    cta_m[threadIdx.x] = top;
    cta_l[threadIdx.x] = total;
  }
#pragma unroll
  for (int j = 0; j < kTilesV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      part[(warp * kKvTokenRows + g + 8 * (i >> 1)) * kRowFloats + kValueBytes * (2 * t + (i & 1)) + j] = o[j][i];
  __syncthreads();
  constexpr int kItems = kKvTokenRows * kD / 4;           // of four columns
  for (int i = threadIdx.x; i < kItems; i += kKvTokenThreads) {
    const int r = i / (kD / 4), d = 4 * (i % (kD / 4));
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kKvTokenWarps; ++w) {
      const float f = row_factor[w][r];
      const float4 v = *reinterpret_cast<const float4*>(part + (w * kKvTokenRows + r) * kRowFloats + d);
      sum.x += f * v.x;
      sum.y += f * v.y;
      sum.z += f * v.z;
      sum.w += f * v.w;
    }
    *reinterpret_cast<float4*>(part + r * kRowFloats + d) = sum;     // over warp 0's, which this thread alone reads here
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  // every CTA finishes a share of the rows' columns
  const int share = (kItems + static_cast<int>(splits) - 1) / static_cast<int>(splits);
  for (int i = static_cast<int>(rank) * share + threadIdx.x; i < min(kItems, (static_cast<int>(rank) + 1) * share); i += kKvTokenThreads) {
    const int r = i / (kD / 4), d = 4 * (i % (kD / 4));
    if (r >= rows || d >= D) continue;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float total = 0.0f;
    if (splits == 1) {
      sum = *reinterpret_cast<const float4*>(part + r * kRowFloats + d);
      total = cta_l[r];
    } else {
      float top = -INFINITY;
      for (uint32_t c = 0; c < splits; ++c) top = fmaxf(top, ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_m[r]), c)));
      for (uint32_t c = 0; c < splits; ++c) {
        const float cm = ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_m[r]), c)), cl = ld_shared_cluster_f32(mapa_cluster(smem_u32(&cta_l[r]), c));
        const float f = cm == -INFINITY ? (cl != cl ? 1.0f : 0.0f) : exp2_ftz(cm - top);
        const float4 v = ld_shared_cluster_f4(mapa_cluster(smem_u32(part + r * kRowFloats + d), c));
        sum.x += f * v.x;
        sum.y += f * v.y;
        sum.z += f * v.z;
        sum.w += f * v.w;
        total += f * cl;
      }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int all = first_row + r;
    T* p = static_cast<T*>(args.out) + (row0 + all / args.group) * args.out_token + (head * args.group + all % args.group) * args.out_head + d;
    if (args.out_vec >= 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T, false>(sum.x * inv, sum.y * inv), pack2<T, false>(sum.z * inv, sum.w * inv));
    } else {
      p[0] = static_cast<T>(sum.x * inv);
      p[1] = static_cast<T>(sum.y * inv);
      p[2] = static_cast<T>(sum.z * inv);
      p[3] = static_cast<T>(sum.w * inv);
    }
  }
  if (splits > 1) cluster_sync();                         // nobody leaves while others read its sums
}

}  // namespace tb200
