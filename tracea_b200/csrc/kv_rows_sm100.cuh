// Attention over the cache for many rows a sequence: prompts.
//
// A CTA takes 256 rows -- tokens times the heads of q that share a head of keys -- as two tiles of 128, and walks over the tokens that
// they see 128 at a time. Both products run on the tcgen05 tensor cores:
//
//   S = q k^^T   128 x 128, q and k^ from shared memory        O += P v^   128 x D, P from tensor memory, v^ from shared memory
//
// Bound by the matrix instructions, 4 rows tokens D operations, and as much by the exponentials, of which an SM does 16 a cycle: two
// tiles of 128 tokens take 2048 cycles of either at D = 128. So the tiles alternate: while one's softmax runs, the other's products
// do. The elements of the cache are widened from e4m3 to halves, exactly, by warps of their own, once for both tiles; a row of q is a
// thread's, scaled into halves on the way in. The weights P lie over the scores' columns, as halves. The pages' scales are applied to
// scores and weights (kv_attention_sm100.cuh).
//
// Tensor memory: 2 x 128 columns of scores (and weights), 2 x 128 of results: all 512. Per step of 128 tokens and tile the issuer's
// order is O += P v^, then the next S over the same P: an S that is complete says that the product in front of it is, and so that O may
// be rescaled.
#pragma once
#include "kv_attention_sm100.cuh"

namespace tb200 {

constexpr int kKvRowsTile = 128, kKvRowsTokens = 128;
constexpr int kKvRowsOfCta = 2 * kKvRowsTile;
constexpr int kKvRowsThreads = 512;            // warps 0..3 and 4..7 softmax of the two tiles, 8..11 widen, 12 issues the products
constexpr int kKvRowsSoftmaxRegs = 176, kKvRowsWidenRegs = 104, kKvRowsMmaRegs = 56;
static_assert(2 * kKvRowsSoftmaxRegs + kKvRowsWidenRegs + kKvRowsMmaRegs <= 4 * 128, "what the block is launched with, 128 a thread");
constexpr int kKvRowsWidenWarp = 8, kKvRowsMmaWarp = 12;
constexpr int kKvRowsMeta = 4;                 // steps whose scales are kept: a softmax is at most two steps behind the widening warps

template <int kD>
__host__ __device__ constexpr int kv_rows_smem_bytes() {
  // q of both tiles, two stages of keys and of values, scales, barriers
  return 1024 + 6 * 128 * kD * 2 + kKvRowsMeta * 8 * 16 + 256;
}

// [q of tile 0, of tile 1][keys, 2 stages][values, 2 stages][scales][barriers]: operands as blocks of 64 columns, 128 rows of 128
// bytes each, swizzled.
template <typename T, int kD>
__global__ void __launch_bounds__(kKvRowsThreads, 1) kv_rows_kernel(const __grid_constant__ KvAttentionArgs args) {
  using namespace ptx;
  constexpr uint32_t kOperand = 128u * kD * 2u, kBlock = 128u * 128u;
  constexpr int kBlocks = kD / 64;
  constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);          // 8-row groups 1024 bytes apart, 128-byte swizzle
  constexpr uint32_t kIdescS = make_idesc(0, 128, 128), kIdescO = make_idesc(0, 128, kD, 1);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = __shfl_sync(0xffffffffu, (smem_u32(smem_raw) + 1023u) & ~1023u, 0);
  uint8_t* const smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t q_smem = smem_base, k_smem = smem_base + 2 * kOperand, v_smem = smem_base + 4 * kOperand;
  float4* const meta = reinterpret_cast<float4*>(smem_gen + 6 * kOperand);      // {keys' scale, values' exponent, 2^-that, -} of 16 tokens
  const uint32_t bars = smem_base + 6 * kOperand + kKvRowsMeta * 8 * 16;
  auto bar = [&](int i) { return bars + 8u * i; };
  constexpr int kQFull = 0, kSFull = 2, kPFull = 4, kOFull = 6, kKFull = 8, kKEmpty = 10, kVFull = 12, kVEmpty = 14, kMetaFull = 16, kDrain = 20, kPFirst = 21;
  volatile uint32_t* const tmem_slot_p = reinterpret_cast<volatile uint32_t*>(smem_gen + 6 * kOperand + kKvRowsMeta * 8 * 16 + 8 * 24);
  volatile uint32_t* const abort_p = tmem_slot_p + 1;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  griddep_launch_dependents();
  griddep_wait();
  const int head = static_cast<int>(blockIdx.x) % args.cache.heads;
  SequenceItem at;
  const int group = args.group;
  if (!find_sequence(args.seqs, static_cast<int>(blockIdx.x) / args.cache.heads, at, [&](int n, int) {
        const long long all = static_cast<long long>(n) * group;
        return all < args.fewest || all > args.most ? 0 : static_cast<int>((all + kKvRowsOfCta - 1) / kKvRowsOfCta);
      }))
    return;
  const int all_rows = at.rows * group;
  const int last_item = (all_rows + kKvRowsOfCta - 1) / kKvRowsOfCta - 1;
  const int first_row = (last_item - at.item) * kKvRowsOfCta;       // the last rows see most: they come first
  const int rows = min(kKvRowsOfCta, all_rows - first_row), tiles = rows > kKvRowsTile ? 2 : 1;
  const int D = args.cache.D, shift = args.cache.page_shift;
  const int begin = at.length - at.rows;
  const int pos_lo = begin + first_row / group, pos_hi = begin + (first_row + rows - 1) / group;
  const int see_lo = args.window > 0 ? max(0, pos_lo - args.window + 1) : 0;
  const int see_hi = min(args.causal ? max(0, pos_hi + 1) : at.length, args.seqs.table_width << shift);
  const int step_lo = see_lo / kKvRowsTokens;
  const int steps = max(0, (see_hi + kKvRowsTokens - 1) / kKvRowsTokens - step_lo);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kQFull + i), kKvRowsTile);
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kPFull + i), kKvRowsTile);
      mbar_init(bar(kPFirst + i), kKvRowsTile);
      mbar_init(bar(kOFull + i), 1);
      mbar_init(bar(kKFull + i), 128);
      mbar_init(bar(kKEmpty + i), 1);
      mbar_init(bar(kVFull + i), 128);
      mbar_init(bar(kVEmpty + i), 1);
    }
    for (int i = 0; i < kKvRowsMeta; ++i) mbar_init(bar(kMetaFull + i), 1);
    mbar_init(bar(kDrain), 1);
    *abort_p = 0u;
    fence_mbar_init();
  }
  if (warp == kKvRowsMmaWarp) {
    tmem_alloc<512>(bars + 8 * 24);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot_p, 0);

  if (warp < kKvRowsWidenWarp) {
    regs_up<kKvRowsSoftmaxRegs>();
    // ------------------------------------------------------------ softmax: a thread a row
    const int tile = warp >> 2, r = (warp & 3) * 32 + lane, my_row = tile * kKvRowsTile + r;
    if (tile < tiles) {
      const bool live = my_row < rows;
      const int token = live ? (first_row + my_row) / group : 0, q_head = head * group + (live ? (first_row + my_row) % group : 0);
      // q into halves, 64 columns at a time. The row is read twice: its largest value is needed first.
      const T* const qp = static_cast<const T*>(args.q) + static_cast<long long>(at.first_row + token) * args.q_token + q_head * args.q_head;
      auto read8 = [&](int d, float(&v)[8]) {
        if (!live || d >= D) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        } else if (args.q_vec) {
          load8(qp + d, v);
        } else {
          load8_upto(qp + d, 1, 8, v);
        }
      };
      float peak = 0.0f;
#pragma unroll
      for (int d = 0; d < kD; d += 8) {
        float v[8];
        read8(d, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) peak = fmaxf(peak, fabsf(v[i]));
      }
      float back;
      const float up = args.sign * row_scale(peak, back);
      const float factor = fmaxf(back * args.scale_log2, 1.17549435e-38f);     // not 0: a score of -infinity stays one
#pragma unroll
      for (int d = 0; d < kD; d += 8) {
        float v[8];
        read8(d, v);
        st_shared_v4(q_smem + tile * kOperand + (d / 64) * kBlock + r * 128 + ((((d % 64) / 8) ^ (r & 7)) * 16),
                     make_uint4(pack_halves(v[0] * up, v[1] * up), pack_halves(v[2] * up, v[3] * up), pack_halves(v[4] * up, v[5] * up),
                                pack_halves(v[6] * up, v[7] * up)));
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(kQFull + tile));

      const int pos = begin + token;
      const int lo = live && args.window > 0 ? pos - args.window + 1 : 0;
      const int hi = !live ? 0x7fffffff : args.causal ? pos + 1 : 0x7fffffff;      // and see_hi, below
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_tmem = tmem + lanes + tile * 128, o_tmem = tmem + lanes + 256 + tile * 128;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        const int t0 = (step_lo + j) * kKvRowsTokens;
        const float4* const scales = meta + (j % kKvRowsMeta) * 8;
        ok = mbar_wait_bounded(bar(kMetaFull + j % kKvRowsMeta), (j / kKvRowsMeta) & 1, abort_p, args.wait_limit) &&
             mbar_wait_bounded(bar(kSFull + tile), j & 1, abort_p, args.wait_limit);
        if (__any_sync(0xffffffffu, !ok)) {
          if (lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, static_cast<uint32_t>(j));
          ok = false;
          break;
        }
        tc_fence_after();
        // columns of this step that the row sees
        const int from = lo - t0, to = min(hi, see_hi) - t0;
        const bool masked = __any_sync(0xffffffffu, from > 0 || to < kKvRowsTokens);
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_tmem + 32 * c, s[c]);
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int i = 0; i < kKvRowsTokens; ++i)
            if (i < from || i >= to) s[i / 32][i % 32] = __float_as_uint(-INFINITY);
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t* const v = s[g / 2] + 16 * (g % 2);
          float gm = __uint_as_float(v[0]);
#pragma unroll
          for (int i = 1; i + 1 < 16; i += 2) gm = max_3(gm, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          gm = fmaxf(gm, __uint_as_float(v[15]));
          const float4 sc = scales[g];
          top = fmaxf(top, gm * (factor * sc.x) + sc.y);
        }
        if (__any_sync(0xffffffffu, top > m + kSlack)) {
          const float next = fmaxf(m, top);
          const float shrink = next == m ? 1.0f : exp2_ftz(m - next);
          m = next;
          l *= shrink;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < kD; c += 16) {
              uint32_t o[16];
              tmem_ld_32x16(o_tmem + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
              tmem_st_32x16(o_tmem + c, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;                // a row that has seen nothing
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float4 sc = scales[2 * c + g];
            const float mul = factor * sc.x, add = sc.y - base;
            const uint64_t mul2 = pack_f32x2(mul, mul), add2 = pack_f32x2(add, add);
            uint64_t sum = 0;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float x, y;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[c][16 * g + i]), __uint_as_float(s[c][16 * g + i + 1])), mul2, add2), x, y);
              x = exp2_ftz(x);
              y = exp2_ftz(y);
              sum = add_f32x2(sum, pack_f32x2(x, y));
              p[8 * g + i / 2] = pack_halves(x, y);
            }
            float x, y;
            unpack_f32x2(sum, x, y);
            l += (x + y) * sc.z;
          }
          tmem_st_32x16(s_tmem + 16 * c, p);
          if (c % 2 == 1) {                                          // half of the weights: the product may begin
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar((c == 1 ? kPFirst : kPFull) + tile));
          }
        }
      }
      // results
      if (ok && steps > 0) {
        ok = mbar_wait_bounded(bar(kOFull + tile), 0, abort_p, args.wait_limit);
        if (__any_sync(0xffffffffu, !ok)) {
          if (lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, 0xffffu);
          ok = false;
        }
      }
      if (ok) {
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* const op = static_cast<T*>(args.out) + static_cast<long long>(at.first_row + token) * args.out_token + q_head * args.out_head;
#pragma unroll
        for (int c = 0; c < kD; c += 32) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld_32x32(o_tmem + c, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int d = 0; d < 32; d += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = l == 0.0f ? 0.0f : __uint_as_float(o[d + i]) * inv;
            if (live && c + d < D) {
              if (args.out_vec == 8) store8(op + c + d, v);
              else store8_upto(op + c + d, 1, 8, v);
            }
          }
        }
      }
    }
  } else if (warp < kKvRowsMmaWarp) {
    regs_down<kKvRowsWidenRegs>();
    // ------------------------------------------------------------ the cache's elements into halves
    const int w = warp - kKvRowsWidenWarp;
    constexpr int kLoads = kD / 16;                                  // of 16 bytes a thread, of keys and of values each
    constexpr int kRowsOfLoad = 2048 / kD;                           // that the four warps cover at once
    // a quarter warp's eight stores of one kind go to two rows of different parity, whose swizzles differ in bit 0: no bank twice
    const int my_row = kD == 128 ? 4 * w + 2 * (lane >> 4) + ((lane >> 2) & 1) : 8 * w + (lane >> 2);
    const int my_block = kD == 128 ? (lane >> 3) & 1 : 0, my_unit = 2 * (lane & 3), my_col = 64 * my_block + 8 * my_unit;
    const long long page_bytes = (static_cast<long long>(args.cache.heads) << shift) * D;
    const long long head_bytes = (static_cast<long long>(head) << shift) * D;
    uint4 kr[kLoads], vr[kLoads];
    int ids = -1, next_ids = -1;                                     // of lane i < 8: page of tokens 16 i .. of a step
    float4 scale;
    auto load_ids = [&](int j) {
      const int token = (step_lo + j) * kKvRowsTokens + 16 * (lane & 7);
      int id = -1;
      if (j < steps && token < see_hi) id = args.seqs.table[at.sequence * args.seqs.table_stride + (token >> shift)];
      return id >= 0 && id < args.cache.pages ? id : -1;
    };
    auto load_scales = [&] {
      scale = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);              // of a page that is not there: weights of 0
      if (w == 0 && ids >= 0) {
        const long long block = static_cast<long long>(ids) * args.cache.heads + head;
        const int ek = static_cast<int>(args.cache.k_scales[block]) - 127, ev = static_cast<int>(args.cache.v_scales[block]) - 127;
        scale = make_float4(power_of_two(ek), static_cast<float>(ev), power_of_two(-ev), 0.0f);
      }
    };
    auto fetch = [&](const uint8_t* from, int j, uint4(&raw)[kLoads]) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = kRowsOfLoad * i + my_row, token = (step_lo + j) * kKvRowsTokens + row;
        const int id = __shfl_sync(0xffffffffu, ids, row >> 4);
        const bool here = id >= 0 && my_col < D && token < see_hi && token >= see_lo;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (here)
          raw[i] = *reinterpret_cast<const uint4*>(from + id * page_bytes + head_bytes +
                                                   static_cast<long long>(token & ((1 << shift) - 1)) * D + my_col);
      }
    };
    auto widen = [&](uint32_t dst, const uint4(&raw)[kLoads]) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = kRowsOfLoad * i + my_row;
        const uint32_t line = dst + my_block * kBlock + row * 128;
        const uint4 x = raw[i];
        uint4 first, second;
        halves_of_e4m3(x.x, first.x, first.y);
        halves_of_e4m3(x.y, first.z, first.w);
        halves_of_e4m3(x.z, second.x, second.y);
        halves_of_e4m3(x.w, second.z, second.w);
        st_shared_v4(line + ((my_unit ^ (row & 7)) * 16), first);
        st_shared_v4(line + (((my_unit + 1) ^ (row & 7)) * 16), second);
      }
    };
    ids = load_ids(0);
    next_ids = load_ids(1);
    load_scales();
    fetch(args.cache.k, 0, kr);
    fetch(args.cache.v, 0, vr);
    for (int j = 0; j < steps; ++j) {
      if (j == args.test_producer_stop) break;                       // test hook: go silent, leave normally
      const int slot = j & 1;
      const uint32_t free_parity = ((j >> 1) & 1) ^ 1;
      if (j >= 2 && !mbar_wait_bounded(bar(kKEmpty + slot), free_parity, abort_p, args.wait_limit)) {
        report_error_status(args.status, abort_p, kErrProducerWait, static_cast<uint32_t>(j));
        break;
      }
      if (w == 0) {
        if (lane < 8) meta[(j % kKvRowsMeta) * 8 + lane] = scale;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kMetaFull + j % kKvRowsMeta));
      }
      widen(k_smem + slot * kOperand, kr);
      fence_proxy_async_smem();
      mbar_arrive(bar(kKFull + slot));
      ids = next_ids;
      if (j + 1 < steps) {
        load_scales();
        fetch(args.cache.k, j + 1, kr);
      }
      next_ids = load_ids(j + 2);
      if (j >= 2 && !mbar_wait_bounded(bar(kVEmpty + slot), free_parity, abort_p, args.wait_limit)) {
        report_error_status(args.status, abort_p, kErrProducerWait, static_cast<uint32_t>(j));
        break;
      }
      widen(v_smem + slot * kOperand, vr);
      fence_proxy_async_smem();
      mbar_arrive(bar(kVFull + slot));
      if (j + 1 < steps) fetch(args.cache.v, j + 1, vr);
    }
    __syncwarp();
  } else {
    regs_down<kKvRowsMmaRegs>();
  }
  if (warp == kKvRowsMmaWarp) {
    // ------------------------------------------------------------ the products (uniform control flow, one lane issues)
    const uint32_t issue = elect_one_lane();
    bool ok = true;
    auto wait = [&](int b, uint32_t parity, int j) {
      ok = ok && mbar_wait_bounded_uniform(bar(b), parity, abort_p, args.wait_limit);
      if (!ok && issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(j));
      return ok;
    };
    auto scores = [&](int tile, int slot) {
      const uint32_t a = (q_smem + tile * kOperand) >> 4, b = (k_smem + slot * kOperand) >> 4;
      mma_step4<false, false>(tmem + tile * 128, a, a + 2, a + 4, a + 6, b, b + 2, b + 4, b + 6, kDescHi, kIdescS, issue);
      if constexpr (kBlocks == 2) {
        const uint32_t a1 = a + (kBlock >> 4), b1 = b + (kBlock >> 4);
        mma_step4<false, true>(tmem + tile * 128, a1, a1 + 2, a1 + 4, a1 + 6, b1, b1 + 2, b1 + 4, b1 + 6, kDescHi, kIdescS, issue);
      }
      tcgen05_commit_if<false>(issue, bar(kSFull + tile));
    };
    for (int tile = 0; tile < tiles && steps > 0; ++tile) {
      if (!wait(kQFull + tile, 0, 0) || (tile == 0 && !wait(kKFull, 0, 0))) break;
      tc_fence_after();
      scores(tile, 0);
    }
    if (ok && steps > 0) tcgen05_commit_if<false>(issue, bar(kKEmpty));
    for (int j = 0; j < steps && ok; ++j) {
      const int slot = j & 1, next = slot ^ 1;
      const uint32_t parity = (j >> 1) & 1, next_parity = ((j + 1) >> 1) & 1;
      for (int tile = 0; tile < tiles; ++tile) {
        if (tile == 0 && !wait(kVFull + slot, parity, j)) break;
        // v^ as it lies, its columns contiguous: 64 of them a block (the leading-dimension offset), 16 tokens 2048 bytes
        const uint32_t b = ((v_smem + slot * kOperand) >> 4) | ((kBlock >> 4) << 16);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait((half == 0 ? kPFirst : kPFull) + tile, j & 1, j)) break;
          tc_fence_after();
#pragma unroll
          for (int k = 4 * half; k < 4 * half + 4; ++k)
            mma_tmem_a_if(issue, tmem + 256 + tile * 128, tmem + tile * 128 + 8 * k, b + 128 * k, kDescHi, kIdescO, j > 0 || k > 0 ? 1u : 0u);
        }
        if (!ok) break;
        if (j + 1 < steps) {
          if (tile == 0 && !wait(kKFull + next, next_parity, j)) break;
          tc_fence_after();
          scores(tile, next);
        } else {
          tcgen05_commit_if<false>(issue, bar(kOFull + tile));
        }
      }
      if (ok) {
        tcgen05_commit_if<false>(issue, bar(kVEmpty + slot));
        if (j + 1 < steps) tcgen05_commit_if<false>(issue, bar(kKEmpty + next));
      }
    }
    // never leave with products under way
    tcgen05_commit_if<false>(issue, bar(kDrain));
    __syncwarp();
    const long long t0 = clock64();
    while (!mbar_try_wait(bar(kDrain), 0) && clock64() - t0 < args.wait_limit) {}
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kKvRowsMmaWarp) tmem_dealloc<512>(tmem);
}

}  // namespace tb200
