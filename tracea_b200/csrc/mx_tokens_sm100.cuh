// The product of mx_gemm_sm100.cuh for few rows: out = epilogue(A W^T), on the same tensor cores with the operands' parts exchanged
// -- 128 rows of W are the rows of an MMA, up to 128 rows of A (tokens) its columns, so that a lone token takes an MMA of 16 columns
// instead of one of 128 rows.
//
// Bound by reading W once, and, as that takes a microsecond or two, by latency: every SM has to take part, and nothing may wait in
// line. A cluster of up to eight CTAs shares 128 rows of W, each a slice of K, whose loads are all in flight at once; the partial
// sums meet in the CTAs' shared memory, always added in the same order, each CTA finishing a share of the outputs.
// kFused: A is still in its storage type and is quantised here, each CTA its slice of K, which saves a launch and a round trip
// through memory in front of a kernel that takes no longer than those.
#pragma once
#include "mx_format.cuh"
#include "mx_gemm_sm100.cuh"

namespace tb200 {

constexpr int kTokMaxRows = 128;
constexpr int kTokThreads = 320;       // warp 0 TMA, warp 1 MMA, warps 2..9 quantise, 2..5 drain the accumulator, 2..9 finish
constexpr int kTokWorkers = 256;
constexpr int kTokMaxStages = 8;
constexpr int kTokBarrierBytes = 256;
constexpr uint32_t kTokWBytes = 128 * kStageKBytes + 2 * kMxTileBytes;      // a k-step of W: codes, scales
constexpr int kTokFusedSteps = 16;     // k-steps of a CTA whose tokens it quantises: they all stay in shared memory

struct MxTokensArgs {
  int M, N, K;                 // tokens, rows of W, columns of both
  int cols;                    // tokens as columns of the MMA: a multiple of 16
  int k_iters;                 // ceil(K / 256)
  int split;                   // CTAs of a cluster
  int num_stages;
  uint32_t idesc;
  const void* x;               // kFused
  long long x_stride;          // elements
  int x_vec;                   // its rows can be read eight elements at a time
  void* out;                   // rows, or codes
  long long out_stride;
  int out_vec;                 // four of its columns are an aligned access
  uint8_t* out_scales;
  int out_blocks, out_k_tiles;
  const void* bias;
  int bias_is_f32;
  const void* residual;
  long long res_stride;
  int act;
  uint32_t* status;
  long long wait_limit;
  int test_producer_stop;
};

__host__ __device__ constexpr uint32_t tok_step_bytes(int cols) { return static_cast<uint32_t>(cols) * kStageKBytes + 2 * kMxTileBytes; }
// [ring: W (and, not fused, the tokens) of every stage][fused: the tokens of every k-step][barriers]. The partial sums, cols x 128
// floats, lie over the front once the accumulator is complete; the barriers are behind them too.
__host__ __device__ constexpr uint32_t tok_front_bytes(int cols, int stages, int fused_steps) {
  const uint32_t ring = static_cast<uint32_t>(stages) * (kTokWBytes + (fused_steps > 0 ? 0u : tok_step_bytes(cols))) +
                        static_cast<uint32_t>(fused_steps) * tok_step_bytes(cols);
  const uint32_t sums = static_cast<uint32_t>(cols) * 512u;
  return ring > sums ? ring : sums;
}
// At least kTokMinSmem: two of these CTAs share an SM's 512 columns of tensor memory; a third, or one of a pair of any other kernel,
// must not come up beside them (see kPairMinSmem).
constexpr int kTokMinSmem = 80 * 1024;
static_assert(3 * (kTokMinSmem + kCtaReservedSmem) > kSmSmemBytes && kTokMinSmem + kPairMinSmem + 2 * kCtaReservedSmem > kSmSmemBytes,
              "clusters with more than an SM's tensor memory");
__host__ __device__ constexpr int tok_smem_bytes(int cols, int stages, int fused_steps) {
  const int n = 1024 + static_cast<int>(tok_front_bytes(cols, stages, fused_steps)) + kTokBarrierBytes;
  return n > kTokMinSmem ? n : kTokMinSmem;
}

template <typename OutT, typename InT, bool kFused, bool kMxOut>
__global__ void __launch_bounds__(kTokThreads, 1)
mx_tokens_sm100_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_sw,
                       const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_sa,
                       const __grid_constant__ MxTokensArgs args) {
  using namespace ptx;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int split = args.split;
  const int rank = static_cast<int>(blockIdx.x) % split, n_tile = static_cast<int>(blockIdx.x) / split;
  const int n0 = n_tile * 128;
  const int m0 = static_cast<int>(blockIdx.y) * kTokMaxRows, tokens = min(kTokMaxRows, args.M - m0);
  const int k_begin = static_cast<int>(static_cast<long long>(args.k_iters) * rank / split);
  const int k_end = static_cast<int>(static_cast<long long>(args.k_iters) * (rank + 1) / split);
  const int steps = k_end - k_begin;
  const uint32_t tok_bytes = tok_step_bytes(args.cols), tok_scales = static_cast<uint32_t>(args.cols) * kStageKBytes;
  const uint32_t stage_bytes = kTokWBytes + (kFused ? 0u : tok_bytes);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = __shfl_sync(0xffffffffu, (smem_u32(smem_raw) + 1023u) & ~1023u, 0);
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int num_stages = args.num_stages;
  const uint32_t fused_off = static_cast<uint32_t>(num_stages) * stage_bytes;
  const uint32_t bar_off = tok_front_bytes(args.cols, num_stages, kFused ? steps : 0);
  const uint32_t bar_base = smem_base + bar_off;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kTokMaxStages + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * kTokMaxStages);
  const uint32_t tmem_slot = tfull_bar + 8u;
  volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(smem_gen + bar_off + 8u * (2 * kTokMaxStages + 1));
  volatile uint32_t* abort_p = tmem_slot_p + 1;
  constexpr uint32_t kTmemCols = 256;              // up to 128 of accumulator, 16 of scales a stage
  constexpr uint32_t kScaleCols0 = 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(tfull_bar, 1);
    *abort_p = 0u;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_sw);
    // a hint only: whatever an earlier kernel still writes there is read after griddep_wait below
    for (int i = 0; i < min(steps, num_stages); ++i) tma_prefetch_2d(&tmap_w, (k_begin + i) * kStageKBytes, n0);
  }
  if (warp == 1) {
    tmem_alloc<kTmemCols>(tmem_slot);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_p, 0);
  griddep_launch_dependents();
  griddep_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (uniform control flow, one lane issues)
    const uint32_t issue = elect_one_lane();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int it = k_begin; it < k_end; ++it) {
      if (issued == args.test_producer_stop) break;   // test hook: go silent, leave normally
      if (issued >= num_stages && !mbar_wait_bounded_uniform(empty_bar(stage), phase ^ 1u, abort_p, args.wait_limit)) {
        if (issue) report_error_status(args.status, abort_p, kErrProducerWait, static_cast<uint32_t>(it));
        ok = false;
        break;
      }
      const uint32_t full = full_bar(stage), dst = smem_base + static_cast<uint32_t>(stage) * stage_bytes;
      mbar_arrive_expect_tx_if(issue, full, stage_bytes);
      tma_load_2d_if(issue, dst, &tmap_w, full, it * kStageKBytes, n0);
      tma_load_3d_if(issue, dst + 128 * kStageKBytes, &tmap_sw, full, 0, 2 * it, n_tile);
      if constexpr (!kFused) {
        tma_load_2d_if(issue, dst + kTokWBytes, &tmap_a, full, it * kStageKBytes, m0);
        tma_load_3d_if(issue, dst + kTokWBytes + tok_scales, &tmap_sa, full, 0, 2 * it, static_cast<int>(blockIdx.y));
      }
      ++issued;
      if (++stage == num_stages) { stage = 0; phase ^= 1u; }
    }
    // never leave with copies in flight into this CTA's shared memory
    if (ok) {
      const int pending = issued < num_stages ? issued : num_stages;
      if (issued < num_stages) { stage = 0; phase = 1u; }
      for (int i = 0; i < pending; ++i) {
        if (!mbar_wait_bounded_uniform(empty_bar(stage), phase ^ 1u, abort_p, args.wait_limit)) break;
        if (++stage == num_stages) { stage = 0; phase ^= 1u; }
      }
    } else {
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { __nanosleep(1000); }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ scales and MMAs (uniform control flow, one lane issues)
    if constexpr (kFused) asm volatile("bar.sync 1, %0;" ::"n"(kTokWorkers + 32) : "memory");   // the tokens are in shared memory
    const uint32_t issue = elect_one_lane();
    constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kScaleDescHi = (128u >> 4) | (1u << 14);
    const uint32_t idesc0 = args.idesc, idesc2 = args.idesc | (2u << 4) | (2u << 29);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
      if (!mbar_wait_bounded_uniform(full_bar(stage), phase, abort_p, args.wait_limit)) {
        if (issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(it));
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t w = (smem_base + static_cast<uint32_t>(stage) * stage_bytes) >> 4;
      const uint32_t tok = kFused ? (smem_base + fused_off + static_cast<uint32_t>(it) * tok_bytes) >> 4 : w + (kTokWBytes >> 4);
      const uint32_t sw = w + ((128 * kStageKBytes) >> 4), st = tok + (tok_scales >> 4);
      const uint32_t tw = tmem_base + kScaleCols0 + 16u * static_cast<uint32_t>(stage), tt = tw + 8u;
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        tmem_cp_32x128b_if<false>(issue, tw + 4u * k, sw + k * (kMxTileBytes >> 4), kScaleDescHi);
        tmem_cp_32x128b_if<false>(issue, tt + 4u * k, st + k * (kMxTileBytes >> 4), kScaleDescHi);
      }
      mx_mma_stage4_probe<false>(tmem_base, w, tok, kDescHi, idesc0, idesc2, tw, tw + 4u, tt, tt + 4u, empty_bar(stage),
                                 full_bar(stage), phase, it != 0 ? 1u : 0u, issue);
      if (++stage == num_stages) { stage = 0; phase ^= 1u; }
    }
    if (ok && issue) mma_commit(tfull_bar);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ workers
    const int wt = static_cast<int>(threadIdx.x) - 64;
    if constexpr (kFused) {
      // this CTA's columns of the tokens, eight a lane, a warp 256 columns -- a k-step -- of one token, four of these at a time
      const int tasks = steps * tokens;
      for (int task0 = wt >> 5; task0 < tasks; task0 += 4 * (kTokWorkers / 32)) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int task = task0 + u * (kTokWorkers / 32);
          const int tok = task / steps, col = (k_begin + task - tok * steps) * 256 + lane * 8;
          const InT* p = static_cast<const InT*>(args.x) + (m0 + tok) * args.x_stride + col;
          const int count = task < tasks ? min(8, args.K - col) : 0;
          if (args.x_vec && count == 8) load8<InT>(p, v[u]);
          else load8_upto<InT>(p, 1, count, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int task = task0 + u * (kTokWorkers / 32);
          if (task >= tasks) break;
          const int tok = task / steps, it = task - tok * steps;
          uint32_t byte;
          const uint32_t codes = mx_quantize8(v[u], byte);
          // the operand's layout: 128-byte rows, 16-byte pieces exchanged by the row's place among eight
          uint8_t* base = smem_gen + fused_off + static_cast<uint32_t>(it) * tok_bytes;
          const uint32_t piece = static_cast<uint32_t>(lane >> 2) ^ (static_cast<uint32_t>(tok) & 7u);
          *reinterpret_cast<uint32_t*>(base + tok * 128 + piece * 16u + (lane & 3) * 4) = codes;
          if ((lane & 3) == 0)
            base[tok_scales + (lane >> 4) * kMxTileBytes + 16 * (tok & 31) + 4 * (tok >> 5) + ((lane >> 2) & 3)] = static_cast<uint8_t>(byte);
        }
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, %0;" ::"n"(kTokWorkers + 32) : "memory");
    }
    if (warp < 6) {
      const bool ready = mbar_wait_bounded_uniform(tfull_bar, 0u, abort_p, 2 * args.wait_limit);
      if (!ready && lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, blockIdx.x);
      if (ready) {
        // partial sums: [token][row of W], over the ring, which nothing reads or writes any more
        tc_fence_after();
        const int quarter = warp & 3;
        float* part = reinterpret_cast<float*>(smem_gen) + quarter * 32 + lane;
        for (int c = 0; c < args.cols; c += 16) {
          uint32_t v[16];
          tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < tokens) part[(c + j) * 128] = __uint_as_float(v[j]);
        }
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  if (split > 1) cluster_sync();
  else __syncthreads();
  // ------------------------------------------------------------ finish: this CTA's 128 / split rows of W, every token, four rows
  // of one token a thread: the loads of all CTAs' parts are in flight together
  if (warp >= 2 && *abort_p == 0u) {
    const int quads = 32 / split;                      // 4 at least; 8 at least, a block, where the output is quantised
    const int wt = static_cast<int>(threadIdx.x) - 64;
    const int f = rank * 4 * quads + wt % quads * 4;
    const int n = n0 + f;
    float bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bias[j] = 0.0f;
      if (args.bias != nullptr && n + j < args.N)
        bias[j] = args.bias_is_f32 ? ld_global_f32(static_cast<const float*>(args.bias) + n + j)
                                   : OutTraits<OutT>::to_f(static_cast<const OutT*>(args.bias)[n + j]);
    }
    for (int tok0 = 0; tok0 < tokens; tok0 += kTokWorkers / quads) {
      const int tok = tok0 + wt / quads;
      const bool tok_ok = tok < tokens;
      const uint32_t at = smem_base + static_cast<uint32_t>((tok_ok ? tok : 0) * 128 + f) * 4u;
      float4 part[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < split) part[r] = ld_shared_cluster_f4(mapa_cluster(at, static_cast<uint32_t>(r)));
      float v[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
      for (int r = 1; r < 8; ++r) {
        if (r < split) {
          v[0] += part[r].x;
          v[1] += part[r].y;
          v[2] += part[r].z;
          v[3] += part[r].w;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += bias[j];
      if constexpr (!kMxOut) {
        if (!tok_ok) continue;
        if (args.residual != nullptr) {
          const OutT* res = static_cast<const OutT*>(args.residual) + (m0 + tok) * args.res_stride + n;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < args.N) v[j] += OutTraits<OutT>::to_f(res[j]);
        }
        OutT* out = static_cast<OutT*>(args.out) + (m0 + tok) * args.out_stride + n;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = apply_act<sizeof(OutT) == 2>(v[j], args.act);
        if (args.out_vec && n + 4 <= args.N) {
          if constexpr (sizeof(OutT) == 2)
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2<OutT, false>(v[0], v[1]), pack2<OutT, false>(v[2], v[3]));
          else
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < args.N) out[j] = OutTraits<OutT>::from_f(v[j]);
        }
      } else {
        // eight neighbouring threads have the 32 columns of a block
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = n + j < args.N ? apply_act<true>(v[j], args.act) : 0.0f;
        float peak = max_abs3(max_abs3(v[0], v[1], v[2]), v[3], 0.0f);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) peak = max_abs3(peak, __shfl_xor_sync(0xffffffffu, peak, d), 0.0f);
        const uint32_t byte = mx_scale_byte(__float_as_uint(peak));
        const float inv = mx_inverse(byte);
        const float s[8] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, 0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t codes = byte == 255u ? 0u : mx_pack8(s);
        const int blk = n / kMxBlock;
        if (tok_ok) {
          if (blk < args.out_blocks)
            *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(args.out) + (m0 + tok) * (16LL * args.out_blocks) + n / 2) =
                static_cast<uint16_t>(codes);
          // blocks past the last one, up to the end of its word, are 0
          if ((n & 31) == 0) args.out_scales[mx_scale_word(m0 + tok, blk >> 2, args.out_k_tiles) + (blk & 3)] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (split > 1) cluster_sync();          // no CTA leaves while another may still read its partial sums
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<kTmemCols>(tmem_base);
  }
}

}  // namespace tb200
