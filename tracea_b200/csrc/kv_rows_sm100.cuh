// Attention over the cache for many rows a sequence: prompts.
//
// A CTA takes 256 rows -- tokens times the heads of q that share a head of keys -- as two tiles of 128, and walks over the tokens that
// they see 128 at a time. Both products run on the tcgen05 tensor cores:
//
//   S = q k^^T   128 x 128, q and k^ from shared memory        O += P v^   128 x D, P from tensor memory, v^ from shared memory
//
// 4 rows tokens D operations, and an exponential for every row and token, of which an SM does 16 a cycle: two tiles of 128 tokens take
// 2048 cycles of either at D = 128. What holds both up is shared memory: of its 128 bytes a cycle the operands of the products take 256 KB
// a step (128 of q, which every 64 tokens' scores read anew, 64 of keys and 64 of values) and the widened keys and values 64 KB, 2560
// cycles. So everything has to run beside everything else: the tiles alternate, each with a warp of its own that issues its products; the
// elements of the cache are widened from e4m3 to halves, exactly, by warps of their own, once for both tiles, whose loads are a step ahead;
// a row of q, scaled into halves on the way in, is a thread's. The weights P lie over the scores' columns, as halves. The pages' scales are
// applied to scores and weights (kv_attention_sm100.cuh).
//
// Tensor memory, all 512 columns: 128 of results a tile, and 128 of scores, as two buffers for 64 tokens each. A softmax goes from one
// buffer to the other: while it works on 64 tokens, the product of the 64 in front is formed and then the scores of the next but one, over
// these weights.
//
// A prompt of 8192 tokens, 32 heads to 8, D = 128: 561 us in a row on the same inputs, 0.98 PFLOP/s (what the mask leaves counted), and
// 590 - 597 on others each time; 395 without a softmax, of which 75 are the CTAs' beginnings and ends; the widening costs nothing beside
// it. Blocks that take over the work of those not launched yet, with q of the next in before the results of the last go out, were slower
// (560 -> 588): the softmax's registers no longer held what it needs.
#pragma once
#include "kv_attention_sm100.cuh"

namespace tb200 {

constexpr int kKvRowsTile = 128, kKvRowsTokens = 128;
constexpr int kKvRowsOfCta = 2 * kKvRowsTile;
constexpr int kKvRowsThreads = 512;            // warps 0..3 and 4..7 softmax of the two tiles, 8..11 widen, 12 and 13 issue the products
constexpr int kKvRowsSoftmaxRegs = 176, kKvRowsWidenRegs = 104, kKvRowsMmaRegs = 56;
static_assert(2 * kKvRowsSoftmaxRegs + kKvRowsWidenRegs + kKvRowsMmaRegs <= 4 * 128, "what the block is launched with, 128 a thread");
constexpr int kKvRowsWidenWarp = 8, kKvRowsMmaWarp = 12;
constexpr int kTestStopOneWarp = 1 << 16;      // test hook: see tracea_b200_test_hooks
constexpr int kKvRowsMeta = 4;                 // steps whose scales are kept: a softmax is at most three steps behind the widening warps

template <int kD>
__host__ __device__ constexpr int kv_rows_smem_bytes() {
  // q of both tiles, two stages of keys and of values, scales, barriers
  return 1024 + 6 * 128 * kD * 2 + kKvRowsMeta * 8 * 16 + 256;
}

struct KvRowsArgs {
  KvAttentionArgs a;
  int splits;                    // CTAs that share a block of rows, each a part of the tokens
  float* sums;                   // splits > 1: [splits][rows * H][kD] results in the making,
  float2* tops;                  // and [splits][rows * H] of {maximum, denominator}
};

// 256 rows of a sequence and a head of keys.
struct RowsItem {
  SequenceItem at;
  int first_row, rows;
};
__device__ __forceinline__ bool rows_item(const KvAttentionArgs& a, int index, RowsItem& item) {
  const int group = a.group;
  if (!find_sequence(a.seqs, index, item.at, [&](int n, int) {
        const long long all = static_cast<long long>(n) * group;
        return all < a.fewest || all > a.most ? 0 : static_cast<int>((all + kKvRowsOfCta - 1) / kKvRowsOfCta);
      }))
    return false;
  const int all_rows = item.at.rows * group, last = (all_rows + kKvRowsOfCta - 1) / kKvRowsOfCta - 1;
  item.first_row = (last - item.at.item) * kKvRowsOfCta;            // the last rows see most: they come first
  item.rows = min(kKvRowsOfCta, all_rows - item.first_row);
  return true;
}

// Whether a row, token `token` of its sequence's in this call, sees a page that is there; `kept`, in shared memory: the sequence, the
// position of its first row, and the tokens that the CTA looks at, from .. to.
__device__ __forceinline__ bool sees_a_page(const KvAttentionArgs& args, uint32_t kept_at, int token) {
  const float4 kept = ptx::ld_shared_f4(kept_at);
  const int p = __float_as_int(kept.y) + token, shift = args.cache.page_shift;
  const int end = args.causal ? min(__float_as_int(kept.w), p + 1) : __float_as_int(kept.w);
  bool sees = false;
  for (int t = max(__float_as_int(kept.z), args.window > 0 ? p - args.window + 1 : 0); t < end && !sees; t = ((t >> shift) + 1) << shift) {
    const int id = args.seqs.table[__float_as_int(kept.x) * args.seqs.table_stride + (t >> shift)];
    sees = id >= 0 && id < args.cache.pages;
  }
  return sees;
}

// [q of tile 0, of tile 1][keys, 2 stages][values, 2 stages][scales][barriers]: operands as blocks of 64 columns, 128 rows of 128
// bytes each, swizzled.
template <typename T, int kD>
__global__ void __launch_bounds__(kKvRowsThreads, 1) kv_rows_kernel(const __grid_constant__ KvRowsArgs call) {
  using namespace ptx;
  const KvAttentionArgs& args = call.a;
  constexpr uint32_t kOperand = 128u * kD * 2u, kBlock = 128u * 128u;
  constexpr int kBlocks = kD / 64;
  constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);          // 8-row groups 1024 bytes apart, 128-byte swizzle
  constexpr uint32_t kIdescS = make_idesc(0, 128, 64), kIdescO = make_idesc(0, 128, kD, 1);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = __shfl_sync(0xffffffffu, (smem_u32(smem_raw) + 1023u) & ~1023u, 0);
  uint8_t* const smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t q_smem = smem_base, k_smem = smem_base + 2 * kOperand, v_smem = smem_base + 4 * kOperand;
  float4* const meta = reinterpret_cast<float4*>(smem_gen + 6 * kOperand);      // {keys' scale, values' exponent, 2^-that, -} of 16 tokens
  const uint32_t bars = smem_base + 6 * kOperand + kKvRowsMeta * 8 * 16;
  auto bar = [&](int i) { return bars + 8u * i; };
  constexpr int kQFull = 0, kSFull = 2, kPFull = 6, kKFull = 10, kKEmpty = 12, kVFull = 14, kVEmpty = 16, kMetaFull = 18, kDrain = 22;   // S, P: 2 tile + buffer
  volatile uint32_t* const tmem_slot_p = reinterpret_cast<volatile uint32_t*>(smem_gen + 6 * kOperand + kKvRowsMeta * 8 * 16 + 8 * 24);
  volatile uint32_t* const abort_p = tmem_slot_p + 1;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  // Tensor memory first: a dependent grid that is let in before may take the columns and wait for this one.
  if (warp == kKvRowsMmaWarp) {
    tmem_alloc<512>(bars + 8 * 24);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot_p, 0);
  griddep_launch_dependents();
  griddep_wait();
  const int split = static_cast<int>(blockIdx.x) % call.splits, id = static_cast<int>(blockIdx.x) / call.splits;
  const int head = id % args.cache.heads, group = args.group;
  RowsItem item;
  if (!rows_item(args, id / args.cache.heads, item)) {
    if (warp == kKvRowsMmaWarp) tmem_dealloc<512>(tmem);
    return;
  }
  const SequenceItem& at = item.at;
  const int first_row = item.first_row, rows = item.rows, tiles = rows > kKvRowsTile ? 2 : 1;
  const int D = args.cache.D, shift = args.cache.page_shift;
  const int begin = at.length - at.rows;
  const int pos_lo = begin + first_row / group, pos_hi = begin + (first_row + rows - 1) / group;
  const int see_lo = args.window > 0 ? max(0, pos_lo - args.window + 1) : 0;
  const int see_hi = min(args.causal ? max(0, pos_hi + 1) : at.length, args.seqs.table_width << shift);
  const int all_steps = max(0, (see_hi + kKvRowsTokens - 1) / kKvRowsTokens - see_lo / kKvRowsTokens);
  const int step_lo = see_lo / kKvRowsTokens + all_steps * split / call.splits;
  const int steps = see_lo / kKvRowsTokens + all_steps * (split + 1) / call.splits - step_lo;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kPFull + i), kKvRowsTile);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kQFull + i), kKvRowsTile);
      mbar_init(bar(kKFull + i), 128);
      mbar_init(bar(kKEmpty + i), tiles);
      mbar_init(bar(kVFull + i), 128);
      mbar_init(bar(kVEmpty + i), tiles);
    }
    for (int i = 0; i < kKvRowsMeta; ++i) mbar_init(bar(kMetaFull + i), 1);
    mbar_init(bar(kDrain), 1);
    mbar_init(bar(kDrain + 1), 1);
    *abort_p = 0u;
    st_shared_v4(bars + 8 * 26, make_uint4(at.sequence, begin, step_lo * kKvRowsTokens, min(see_hi, (step_lo + steps) * kKvRowsTokens)));
    fence_mbar_init();
  }
  __syncthreads();

  if (warp < kKvRowsWidenWarp) {
    regs_up<kKvRowsSoftmaxRegs>();
    // ------------------------------------------------------------ softmax: a thread a row
    const int tile = warp >> 2, r = (warp & 3) * 32 + lane, my_row = tile * kKvRowsTile + r;
    if (tile < tiles) {
      const bool live = my_row < rows;
      const int token = live ? (first_row + my_row) / group : 0, q_head = head * group + (live ? (first_row + my_row) % group : 0);
      // q into halves: kD / 8 lanes a row, eight columns each, all of the warp's rows' loads under way together
      constexpr int kRowLanes = kD / 8, kRowsAtOnce = 32 / kRowLanes, kLoads = kRowLanes;
      const int col = 8 * (lane % kRowLanes), first = tile * kKvRowsTile + (warp & 3) * 32 + lane / kRowLanes;
      const T* const q0 = static_cast<const T*>(args.q) + static_cast<long long>(at.first_row) * args.q_token + head * group * args.q_head + col;
      Vec8<T> raw[kLoads];
      auto load_rows = [&](auto fetch_row) {
        // a division for the first row's token and head, steps from there
        const int step_token = kRowsAtOnce / group, step_head = kRowsAtOnce % group;
        int q_tok = (first_row + first) / group, q_sub = (first_row + first) % group;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          raw[i] = Vec8<T>{};
          if (col < D && first + i * kRowsAtOnce < rows) fetch_row(q0 + q_tok * args.q_token + q_sub * args.q_head, raw[i]);
          q_tok += step_token;
          q_sub += step_head;
          if (q_sub >= group) {
            q_sub -= group;
            ++q_tok;
          }
        }
      };
      if (args.q_vec) {
        load_rows([](const T* p, Vec8<T>& v) { fetch8(p, v); });
      } else {
        load_rows([](const T* p, Vec8<T>& v) {
#pragma unroll
          for (int k = 0; k < 8; ++k) reinterpret_cast<T*>(&v)[k] = p[k];
        });
      }
      // Peaks of the rows: every exchange halves the rows that a lane holds, until lane i of a row's lanes has that of load i.
      float peak[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        float v[8];
        widen8(raw[i], v);
        peak[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) peak[i] = fmaxf(peak[i], fabsf(v[k]));
      }
#pragma unroll
      for (int o = kRowLanes / 2; o > 0; o >>= 1) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? peak[i] : peak[i + o], o);
          peak[i] = fmaxf(upper ? peak[i + o] : peak[i], other);
        }
      }
      float back;
      const float up_of_lane = args.sign * row_scale(peak[0], back);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int in_tile = (warp & 3) * 32 + i * kRowsAtOnce + lane / kRowLanes;
        const float up = __shfl_sync(0xffffffffu, up_of_lane, i, kRowLanes);
        float v[8];
        widen8(raw[i], v);
        st_shared_v4(q_smem + tile * kOperand + (col / 64) * kBlock + in_tile * 128 + ((((col % 64) / 8) ^ (in_tile & 7)) * 16),
                     make_uint4(pack_halves(v[0] * up, v[1] * up), pack_halves(v[2] * up, v[3] * up), pack_halves(v[4] * up, v[5] * up),
                                pack_halves(v[6] * up, v[7] * up)));
      }
      // This thread's row is row lane / kRowsAtOnce of the loads. Times a page's scale, 2^-40 or more, it must not vanish: masked scores are
      // -infinity before that product. Where 2^-86 is more than the row's own factor, scores, which are below 2^17 2^40 times it, move by
      // less than 2^-29.
      const float factor = fmaxf(__shfl_sync(0xffffffffu, back, (lane % kRowsAtOnce) * kRowLanes + lane / kRowsAtOnce) * args.scale_log2, 0x1p-86f);
      fence_proxy_async_smem();
      mbar_arrive(bar(kQFull + tile));

      const int pos = begin + token;
      const int lo = live && args.window > 0 ? pos - args.window + 1 : 0;
      const int hi = !live ? 0x7fffffff : args.causal ? pos + 1 : 0x7fffffff;      // and see_hi, below
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_tmem = tmem + lanes + tile * 128, o_tmem = tmem + lanes + 256 + tile * 128;
      float m = -INFINITY, l = 0.0f;
      bool ok = true, far = false;                                   // far: a maximum of the warp's rows is (kFar)
      auto wait_scores = [&](int h) {                                // of half step h; it says too that the product of h - 2 is complete
        ok = mbar_wait_bounded(bar(kSFull + 2 * tile + (h & 1)), (h >> 1) & 1, abort_p, args.wait_limit);
        if (__any_sync(0xffffffffu, !ok)) {
          if (lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, static_cast<uint32_t>(h));
          ok = false;
        }
        tc_fence_after();
        return ok;
      };
      for (int h = 0; h < 2 * steps; ++h) {
        const int j = h >> 1, t0 = (step_lo + j) * kKvRowsTokens + 64 * (h & 1);
        const uint32_t buffer = s_tmem + 64 * (h & 1);
        const float4* const scales = meta + (j % kKvRowsMeta) * 8 + 4 * (h & 1);
        if (!wait_scores(h)) break;
        uint32_t s[2][32];
        tmem_ld_32x32(buffer, s[0]);
        tmem_ld_32x32(buffer + 32, s[1]);
        // columns that the row sees
        const int from = lo - t0, to = min(hi, see_hi) - t0;
        const bool masked = __any_sync(0xffffffffu, from > 0 || to < 64);
        ok = mbar_wait_bounded(bar(kMetaFull + j % kKvRowsMeta), (j / kKvRowsMeta) & 1, abort_p, args.wait_limit);
        if (__any_sync(0xffffffffu, !ok)) {
          if (lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, static_cast<uint32_t>(h));
          ok = false;
          break;
        }
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i < from || i >= to) s[i / 32][i % 32] = __float_as_uint(-INFINITY);
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t* const v = s[g / 2] + 16 * (g % 2);
          float gm = __uint_as_float(v[0]);
#pragma unroll
          for (int i = 1; i + 1 < 16; i += 2) gm = max_3(gm, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          gm = fmaxf(gm, __uint_as_float(v[15]));
          const float4 sc = scales[g];
          top = fmaxf(top, fmaf(gm, factor * sc.x, sc.y));
        }
        if (far || __any_sync(0xffffffffu, top > m + kSlack)) {
          const float next = fmaxf(m, top);
          far = __any_sync(0xffffffffu, is_far(next));
          const float shrink = next == m ? 1.0f : exp2_ftz(m - next);
          m = next;
          l *= shrink;
          if (h > 0) {
            if (!wait_scores(h + 1)) break;                          // the product of h - 1 is complete
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
        auto weights = [&](auto is_far_form) {
          constexpr bool kFarForm = decltype(is_far_form)::value;
          const float base = m == -INFINITY ? 0.0f : kFarForm ? m : m - kLift;         // 0: a row that has seen nothing
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float4 sc = scales[2 * c + g];
              const float mul = factor * sc.x, add = kFarForm ? sc.y : sc.y - base;
              const uint64_t mul2 = pack_f32x2(mul, mul), add2 = pack_f32x2(add, add);
              uint64_t sum = 0;
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float x, y;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[c][16 * g + i]), __uint_as_float(s[c][16 * g + i + 1])), mul2, add2), x, y);
                if constexpr (kFarForm) {        // the score, then what it is from the maximum, then the lift
                  x = x - base + kLift;
                  y = y - base + kLift;
                }
                x = exp2_ftz(x);
                y = exp2_ftz(y);
                sum = add_f32x2(sum, pack_f32x2(x, y));
                p[8 * g + i / 2] = pack_halves(x, y);
              }
              float x, y;
              unpack_f32x2(sum, x, y);
              l += (x + y) * sc.z;
            }
            tmem_st_32x16(buffer + 16 * c, p);
          }
        };
        if (far) weights(std::true_type{});
        else weights(std::false_type{});
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar(kPFull + 2 * tile + (h & 1)));
      }
      // results
      if (ok && steps > 0) wait_scores(2 * steps + 1);               // the last product is complete
      if (ok) {
        tc_fence_after();
        // A row of q that is not finite takes NaN from pages that are not there, too, whose scores no mask hides; it is NaN only if it sees
        // a token. (m is -infinity as long as all scores are NaN or of such pages. What this takes waits in shared memory: no register is
        // left for it.)
        if (live && m == -INFINITY && l != l && !sees_a_page(args, bars + 8 * 26, token)) l = 0.0f;
        const bool whole = call.splits == 1;
        const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        T* const op = static_cast<T*>(args.out) + static_cast<long long>(at.first_row + token) * args.out_token + q_head * args.out_head;
        const long long heads = static_cast<long long>(args.cache.heads) * group;
        const long long part = (split * static_cast<long long>(args.seqs.rows) + at.first_row + token) * heads + q_head;
        if (!whole && live) call.tops[part] = make_float2(m, l);
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
              if (!whole) store8(call.sums + part * kD + c + d, v);
              else if (args.out_vec == 8) store8(op + c + d, v);
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
    // Places and scales are loaded steps ahead and looked at only when they are needed: what looks at a load waits for it.
    int ids = -1, next_ids = -1;                                     // of lane i < 8: page of tokens 16 i .. of a step
    uint32_t k_byte = 0, v_byte = 0;                                 // its scales
    auto load_ids = [&](int j) {
      const int token = (step_lo + j) * kKvRowsTokens + 16 * (lane & 7);
      return j < steps && token < see_hi ? args.seqs.table[at.sequence * args.seqs.table_stride + (token >> shift)] : -1;
    };
    auto there = [&](int id) { return id >= 0 && id < args.cache.pages; };
    auto load_scales = [&] {
      if (w == 0 && there(ids)) {
        const long long block = static_cast<long long>(ids) * args.cache.heads + head;
        k_byte = args.cache.k_scales[block];
        v_byte = args.cache.v_scales[block];
      }
    };
    auto put_scales = [&](int j) {
      float4 scale = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);       // of a page that is not there: weights of 0
      if (there(ids)) {
        const int ek = static_cast<int>(k_byte) - 127, ev = static_cast<int>(v_byte) - 127;
        scale = make_float4(power_of_two(ek), static_cast<float>(ev), power_of_two(-ev), 0.0f);
      }
      if (lane < 8) meta[(j % kKvRowsMeta) * 8 + lane] = scale;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kMetaFull + j % kKvRowsMeta));
    };
    auto fetch = [&](const uint8_t* from, int j, uint4(&raw)[kLoads]) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = kRowsOfLoad * i + my_row, token = (step_lo + j) * kKvRowsTokens + row;
        const int id = __shfl_sync(0xffffffffu, ids, row >> 4);
        const bool here = there(id) && my_col < D && token < see_hi && token >= see_lo;
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
    fetch(args.cache.v, 0, vr);
    fetch(args.cache.k, 0, kr);
    bool ok = true;
    // For slot j % 2 to be free of step j - 2. The whole warp goes on or gives up: what follows exchanges values between its lanes.
    auto wait = [&](int b, int j) {
      if (j >= 2 && !mbar_wait_bounded_uniform(bar(b + (j & 1)), ((j >> 1) & 1) ^ 1, abort_p, args.wait_limit)) {
        if (lane == 0) report_error_status(args.status, abort_p, kErrProducerWait, static_cast<uint32_t>(j));
        ok = false;
      }
      return ok;
    };
    // keys, and the scales, a step ahead of the values: ids and scale are those of keys' step j
    for (int j = 0; j <= steps && ok; ++j) {
      // test hook: all four warps, or the last of them alone, go silent and leave normally
      if (j == args.test_producer_stop || (w == 3 && j + kTestStopOneWarp == args.test_producer_stop)) break;
      if (j < steps) {
        if (!wait(kKEmpty, j)) break;
        if (w == 0) put_scales(j);
        widen(k_smem + (j & 1) * kOperand, kr);
        fence_proxy_async_smem();
        mbar_arrive(bar(kKFull + (j & 1)));
      }
      if (j > 0) {
        if (!wait(kVEmpty, j - 1)) break;
        widen(v_smem + ((j - 1) & 1) * kOperand, vr);
        fence_proxy_async_smem();
        mbar_arrive(bar(kVFull + ((j - 1) & 1)));
        if (j < steps) fetch(args.cache.v, j, vr);
      }
      ids = next_ids;
      if (j + 1 < steps) {
        load_scales();
        fetch(args.cache.k, j + 1, kr);
      }
      next_ids = load_ids(j + 2);
    }
    __syncwarp();
  } else {
    regs_down<kKvRowsMmaRegs>();
  }
  if (warp >= kKvRowsMmaWarp && warp < kKvRowsMmaWarp + tiles) {
    // ------------------------------------------------------------ a tile's products (uniform control flow, one lane issues)
    const uint32_t issue = elect_one_lane();
    const int tile = warp - kKvRowsMmaWarp;
    bool ok = true;
    auto wait = [&](int b, uint32_t parity, int j) {
      ok = ok && mbar_wait_bounded_uniform(bar(b), parity, abort_p, args.wait_limit);
      if (!ok && issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(j));
      return ok;
    };
    // scores of half step h: 64 of the step's 128 rows of keys
    auto scores = [&](int h) {
      const uint32_t a = (q_smem + tile * kOperand) >> 4, b = (k_smem + ((h >> 1) & 1) * kOperand + (h & 1) * (64 * 128)) >> 4;
      const uint32_t d = tmem + tile * 128 + 64 * (h & 1);
      mma_step4<false, false>(d, a, a + 2, a + 4, a + 6, b, b + 2, b + 4, b + 6, kDescHi, kIdescS, issue);
      if constexpr (kBlocks == 2) {
        const uint32_t a1 = a + (kBlock >> 4), b1 = b + (kBlock >> 4);
        mma_step4<false, true>(d, a1, a1 + 2, a1 + 4, a1 + 6, b1, b1 + 2, b1 + 4, b1 + 6, kDescHi, kIdescS, issue);
      }
    };
    if (steps > 0 && wait(kQFull + tile, 0, 0) && wait(kKFull, 0, 0)) {
      tc_fence_after();
      for (int h = 0; h < 2; ++h) {
        scores(h);
        tcgen05_commit_if<false>(issue, bar(kSFull + 2 * tile + h));
      }
      tcgen05_commit_if<false>(issue, bar(kKEmpty));
    }
    for (int h = 0; h < 2 * steps && ok; ++h) {
      const int j = h >> 1, slot = j & 1, next = slot ^ 1;
      if (h % 2 == 0 && !wait(kVFull + slot, (j >> 1) & 1, j)) break;
      if (h % 2 == 0 && j + 1 < steps && !wait(kKFull + next, ((j + 1) >> 1) & 1, j)) break;
      if (!wait(kPFull + 2 * tile + (h & 1), j & 1, j)) break;
      tc_fence_after();
      // v^ as it lies, its columns contiguous: 64 of them a block (the leading-dimension offset), 16 tokens 2048 bytes
      const uint32_t b = ((v_smem + slot * kOperand + (h & 1) * (64 * 128)) >> 4) | ((kBlock >> 4) << 16);
      const uint32_t p = tmem + tile * 128 + 64 * (h & 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_tmem_a_if(issue, tmem + 256 + tile * 128, p + 8 * k, b + 128 * k, kDescHi, kIdescO, h > 0 || k > 0 ? 1u : 0u);
      if (h + 2 < 2 * steps) scores(h + 2);
      tcgen05_commit_if<false>(issue, bar(kSFull + 2 * tile + (h & 1)));         // scores of h + 2, or that there are none
      if (h % 2 == 1) {
        tcgen05_commit_if<false>(issue, bar(kVEmpty + slot));
        if (j + 1 < steps) tcgen05_commit_if<false>(issue, bar(kKEmpty + next));
      }
    }
    // never leave with products under way
    tcgen05_commit_if<false>(issue, bar(kDrain + tile));
    __syncwarp();
    const long long t0 = clock64();
    while (!mbar_try_wait(bar(kDrain + tile), 0) && clock64() - t0 < args.wait_limit) {}
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kKvRowsMmaWarp) tmem_dealloc<512>(tmem);
}

// The sums of rows whose tokens were split: a warp to a row, a CTA to 256 rows as above, a lane four columns.
constexpr int kKvRowsJoinWarps = 8;
template <typename T, int kD>
__global__ void __launch_bounds__(32 * kKvRowsJoinWarps) kv_rows_join_kernel(const __grid_constant__ KvRowsArgs call) {
  using namespace ptx;
  const KvAttentionArgs& args = call.a;
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = static_cast<int>(blockIdx.x), head = id % args.cache.heads, group = args.group;
  RowsItem item;
  if (!rows_item(args, id / args.cache.heads, item)) return;
  const long long heads = static_cast<long long>(args.cache.heads) * group, all = args.seqs.rows * heads;
  for (int r = static_cast<int>(blockIdx.y) * kKvRowsJoinWarps + warp; r < item.rows; r += kKvRowsJoinWarps * static_cast<int>(gridDim.y)) {
    const int row = item.first_row + r, token = item.at.first_row + row / group, q_head = head * group + row % group;
    const long long part = token * heads + q_head;
    float top = -INFINITY, total = 0.0f;
    for (int s = 0; s < call.splits; ++s) top = fmaxf(top, call.tops[s * all + part].x);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < call.splits; ++s) {
      const float2 t = call.tops[s * all + part];
      const float f = part_factor(t.x, t.y, top);
      total += f * t.y;
      if (4 * lane < args.cache.D) add_scaled(sum, *reinterpret_cast<const float4*>(call.sums + (s * all + part) * kD + 4 * lane), f);
    }
    T* const p = static_cast<T*>(args.out) + token * args.out_token + q_head * args.out_head + 4 * lane;
    if (4 * lane < args.cache.D) store_4(p, sum, total == 0.0f ? 0.0f : 1.0f / total, args.out_vec);
  }
}

}  // namespace tb200
