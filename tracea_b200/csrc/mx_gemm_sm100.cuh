// Matrix product of two operands in the 4-bit microscaled format (mx_format.cuh), out = epilogue(A W^T), on the block-scaled tensor
// cores: TMA loads -> smem ring -> tcgen05.cp of the scales into TMEM -> tcgen05.mma kind::mxf4 -> TMEM -> fused epilogue.
//
// A k-step is 128 bytes of each row, 256 columns: four MMAs of 64, each with two scales a row. The scales of 128 rows x 4 blocks
// lie in memory as the 512 bytes that tcgen05.cp spreads over 32 lanes x 4 columns (and repeats for the four lane quarters), so
// a stage's scales are copied by the TMA unit beside its operands and never touched by a thread.
//
// What bounds it: an MMA of M rows x N columns takes N / 2 cycles whatever the format, and 4-bit operands bring four times as
// many products a byte as 16-bit ones -- so a k-step takes as long as a 128-byte k-step of the 16-bit kernel, and the same tilings
// are fed by the same bytes per cycle from L2 (all SMs together get about 87 B/cycle/SM).
#pragma once
#include "mx_format.cuh"

namespace tb200 {

enum : int { kMxStoreTma = 0, kMxStoreRows = 1, kMxStoreMx = 2 };

constexpr int kMxMaxStages = 8;
// Warp 0 TMA, warp 1 MMA, then the epilogue's warps in groups of four, one more TMA, pairs: two for scales. Quantised output has
// four groups, others, whose rows go through 64 registers at a time, two: what bounds an epilogue beside MMAs is the latency
// of its chain of instructions (SiLU into 4 bits, 64 columns: 2050 cycles a warp at two warps a scheduler).
__host__ __device__ constexpr int mx_epilogue_warps(int bn, int store) { return store == kMxStoreMx && bn > 64 ? 16 : 8; }
__host__ __device__ constexpr int mx_threads(int bn, bool pair, int store) { return 32 * ((pair ? 5 : 3) + mx_epilogue_warps(bn, store)); }

struct MxGemmArgs {
  int M, N;
  int k_iters;                 // ceil(K / 256)
  int num_m_tiles, num_n_tiles;
  int panel_width, panel_tiles;
  int num_stages;
  uint32_t idesc;
  void* out;                   // kMxStoreRows, TMA stores go by their map; kMxStoreMx: the codes
  long long out_stride;        // elements
  int out_vec;                 // kMxStoreRows: bytes a lane may store at once
  uint8_t* out_scales;         // kMxStoreMx
  int out_blocks, out_k_tiles;
  const void* bias;
  int bias_is_f32;
  const void* residual;        // same dtype as out
  long long res_stride;
  int res_vec;
  int act;
  uint32_t* status;
  long long wait_limit;
  int test_producer_stop;
};

// Bytes of a stage: rows of A, rows of W, scales of 128 rows of A, scales of the 128-row tiles that the columns touch.
__host__ __device__ constexpr int mx_b_scale_tiles(int bn) { return bn <= 128 ? 1 : 2; }
__host__ __device__ constexpr int mx_stage_bytes(int bn, bool pair) {
  return kBlockM * kStageKBytes + (pair ? bn / 2 : bn) * kStageKBytes + (1 + mx_b_scale_tiles(bn)) * 2 * kMxTileBytes;
}
constexpr int kMxBarrierBytes = 256;
// Boxes of 32 rows x 128 bytes for each epilogue warp. Stages are worth more than a second box where a tile is large.
__host__ __device__ constexpr int mx_staging_depth(int bn, int store) { return store == kMxStoreMx ? 0 : (bn == 256 ? 1 : 2); }
__host__ __device__ constexpr int mx_smem_bytes(int bn, int stages, bool pair, int store) {
  return 1024 + stages * mx_stage_bytes(bn, pair) + mx_epilogue_warps(bn, store) * (mx_staging_depth(bn, store) * kStagingBoxBytes + bn * 4) +
         kMxBarrierBytes;
}

// Tiles of 256 columns leave no room in TMEM for a second accumulator beside the scales.
__host__ __device__ constexpr int mx_accumulators(int bn) { return bn == 256 ? 1 : 2; }
// TMEM columns: one or two accumulators, then the scales of every stage (8 columns of A's, 8 per tile of W's). A stage's columns are
// rewritten when its shared memory is, which the stage's empty barrier orders behind the MMAs that read them.
__host__ __device__ constexpr int mx_scale_cols(int bn) { return 8 + 8 * mx_b_scale_tiles(bn); }
// Pipeline stages: what shared memory holds and tensor memory has columns of scales for.
__host__ __device__ constexpr int mx_num_stages(int bn, bool pair, int store) {
  const int in_smem = (232448 - mx_smem_bytes(bn, 0, pair, store)) / mx_stage_bytes(bn, pair);
  const int in_tmem = (512 - mx_accumulators(bn) * bn) / mx_scale_cols(bn), n = in_smem < in_tmem ? in_smem : in_tmem;
  return n < kMxMaxStages ? n : kMxMaxStages;
}

// apply_act32, but for ReLU, which keeps NaN, and GELU (see kGeluA), with fewer trips through the special-function unit for SiLU: a tile of 192 columns of 1024 takes
// 2200 cycles of MMAs and 128 x 192 exponentials and reciprocals, at 16 of these a cycle, 3100. Four values share a reciprocal,
// 1 / a = (1 / abcd) bcd, which costs three roundings more, 2^-22 -- far below a 16- or 4-bit result's. The product of four stays
// in range while each 1 + e^-x is below 2^31: 32 columns of a row with a value below -20, or a NaN, take the other way. (Each lane
// for itself: rows past M, whose scales are anyone's, must not choose for the others.)
template <bool kFast>
__device__ __forceinline__ void mx_act32(float (&f)[32], int act) {
  if (act == kActRelu) {
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = relu_nan(f[j]);
    return;
  }
  if (kFast && act == kActGelu) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      float a = f[j], b = f[j + 1];
      mul2(a, b, f[j], f[j + 1]);
      fma2(a, b, kGeluB, kGeluB, kGeluA, kGeluA);
      mul2(a, b, f[j], f[j + 1]);
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
      add2(a, b, 1.0f, 1.0f);
      asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
      asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
      mul2(f[j], f[j + 1], a, b);
    }
    return;
  }
  if (!kFast || act != kActSilu) {
    apply_act32<kFast>(f, act);
    return;
  }
  float low = f[0];
#pragma unroll
  for (int j = 1; j < 31; j += 2) low = min_nan3(low, f[j], f[j + 1]);
  low = min_nan3(low, f[31], f[31]);
  if (!(low >= -20.0f)) {
    apply_act32<kFast>(f, act);
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    float a[4] = {f[j], f[j + 1], f[j + 2], f[j + 3]};
    mul2(a[0], a[1], -1.44269504f, -1.44269504f);
    mul2(a[2], a[3], -1.44269504f, -1.44269504f);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a[i]));
    add2(a[0], a[1], 1.0f, 1.0f);
    add2(a[2], a[3], 1.0f, 1.0f);
    float p = a[0], q = a[1], r;
    mul2(p, q, a[2], a[3]);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p * q));
    const float rp = r * q, rq = r * p;       // 1 / (a[0] a[2]), 1 / (a[1] a[3])
    // the reciprocals, at most 1, before the values: a value times a neighbour's denominator may pass fp32's range
    mul2(a[0], a[1], rp, rq);
    mul2(a[2], a[3], rp, rq);
    mul2(f[j], f[j + 1], a[2], a[3]);
    mul2(f[j + 2], f[j + 3], a[0], a[1]);
  }
}

// A warp's box (32 rows of 128 bytes, 16-byte pieces exchanged by the row's place among eight) from and to rows of global memory, in
// accesses of `vec` bytes -- 16, 8, 4 or one element, what all rows allow; `at` is the box's first element, `stride` its rows' pitch
// (`base`: an address that may be read). The residual comes in asynchronously, the boxes all in flight while the accumulator is being
// computed. 1500 x 1030 x 777 in fp32: 7.5 us with a residual that is not in L2 and 7.1 with one that is; with loads through
// registers, four or eight of which were in flight, 11.7 and 8.3.
template <typename OutT, int kBytes>
__device__ __noinline__ void mx_fetch_box(uint32_t stg, const OutT* base, const OutT* at, long long stride, int rows_left, int cols_left, int lane) {
  constexpr int kLanes = 128 / kBytes, kStep = 32 / kLanes;       // lanes of a row, rows of an instruction
  const uint32_t byte = static_cast<uint32_t>(lane % kLanes) * kBytes;
  const bool col_ok = static_cast<int>(byte / sizeof(OutT)) < cols_left;
  int r = lane / kLanes;
  const OutT* src = at + r * stride + (col_ok ? byte / sizeof(OutT) : 0u);
#pragma unroll 8
  for (int i = 0; i < kLanes; ++i) {
    const bool live = col_ok && r < rows_left;
    ptx::cp_async_or_zero<kBytes>(stg + static_cast<uint32_t>(r) * 128u + (((byte >> 4) ^ (static_cast<uint32_t>(r) & 7u)) << 4) + (byte & 15u),
                                  live ? src : base, live);
    src += kStep * stride;
    r += kStep;
  }
}
template <typename OutT, typename Word>
__device__ __noinline__ void mx_store_box(uint32_t stg, OutT* at, long long stride, int rows_left, int cols_left, int lane) {
  constexpr int kBytes = sizeof(Word);
  constexpr int kSegs = kBytes == 2 ? 2 : 1, kLanes = kBytes == 2 ? 32 : 128 / kBytes, kStep = 32 / kLanes;
  __syncwarp();                            // every lane's row is in the box
  const uint32_t byte = static_cast<uint32_t>(lane % kLanes) * kBytes;
  int r = lane / kLanes;
  uint8_t* dst = reinterpret_cast<uint8_t*>(at + r * stride) + byte;
#pragma unroll 8
  for (int i = 0; i < kLanes; ++i) {
#pragma unroll
    for (int s = 0; s < kSegs; ++s) {
      const uint32_t b = byte + s * 64u, from = stg + static_cast<uint32_t>(r) * 128u + (((b >> 4) ^ (static_cast<uint32_t>(r) & 7u)) << 4) + (b & 15u);
      Word w;
      if constexpr (kBytes == 16) w = ptx::ld_shared_v4(from);
      else if constexpr (kBytes == 8) w = ptx::ld_shared_v2(from);
      else w = ptx::ld_shared_word<Word>(from);
      if (static_cast<int>(b / sizeof(OutT)) < cols_left && r < rows_left) *reinterpret_cast<Word*>(dst + s * 64) = w;
    }
    dst += kStep * stride * static_cast<long long>(sizeof(OutT));
    r += kStep;
  }
  __syncwarp();                            // the box may be rewritten once every lane has read it out
}
template <typename OutT>
__device__ __forceinline__ void mx_fetch_rows(int vec, uint32_t stg, const OutT* base, const OutT* at, long long stride, int rows_left, int cols_left, int lane) {
  if (vec == 16) mx_fetch_box<OutT, 16>(stg, base, at, stride, rows_left, cols_left, lane);
  else if (vec == 8) mx_fetch_box<OutT, 8>(stg, base, at, stride, rows_left, cols_left, lane);
  else if (vec == 4) mx_fetch_box<OutT, 4>(stg, base, at, stride, rows_left, cols_left, lane);
  else if constexpr (sizeof(OutT) == 2) coop_load_box_narrow<OutT, uint16_t>(stg, at, lane * stride, lane < rows_left, cols_left, lane);
}
template <typename OutT>
__device__ __forceinline__ void mx_store_rows(int vec, uint32_t stg, OutT* at, long long stride, int rows_left, int cols_left, int lane) {
  if (vec == 16) mx_store_box<OutT, uint4>(stg, at, stride, rows_left, cols_left, lane);
  else if (vec == 8) mx_store_box<OutT, uint2>(stg, at, stride, rows_left, cols_left, lane);
  else if (vec == 4) mx_store_box<OutT, uint32_t>(stg, at, stride, rows_left, cols_left, lane);
  else if constexpr (sizeof(OutT) == 2) mx_store_box<OutT, uint16_t>(stg, at, stride, rows_left, cols_left, lane);
}

template <typename OutT, int BN, bool kPair, int kStore>
__global__ void __launch_bounds__(mx_threads(BN, kPair, kStore), 1)
mx_gemm_sm100_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                     const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sw,
                     const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ MxGemmArgs args) {
  using namespace ptx;
  constexpr uint32_t kABytes = kBlockM * kStageKBytes;
  constexpr uint32_t kBRows = kPair ? BN / 2 : BN;
  constexpr uint32_t kBBytes = kBRows * kStageKBytes;
  constexpr uint32_t kBTiles = mx_b_scale_tiles(BN);
  constexpr uint32_t kSaOff = kABytes + kBBytes, kSbOff = kSaOff + 2 * kMxTileBytes;
  constexpr uint32_t kStageBytes = mx_stage_bytes(BN, kPair);
  constexpr int kTileM = kPair ? 2 * kBlockM : kBlockM;
  constexpr uint32_t kScaleCols = mx_scale_cols(BN);
  constexpr int kStagingDepth = mx_staging_depth(BN, kStore);
  static_assert(BN % 64 == 0 && BN <= 256 && kStageBytes % 1024 == 0, "tile");
  constexpr int kEpiWarps = mx_epilogue_warps(BN, kStore), kEpiGroups = kEpiWarps / 4;
  constexpr int kSecondProducer = 2 + kEpiWarps, kScaleWarp = 3 + kEpiWarps;
  constexpr int kAcc = mx_accumulators(BN);            // the host keeps to as many stages as TMEM has columns of scales for
  constexpr uint32_t kTmemCols = 512;
  const uint32_t cta_rank = kPair ? __shfl_sync(0xffffffffu, cluster_ctarank(), 0) : 0u;
  const bool leader = cta_rank == 0u;
  const int worker = kPair ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_workers = kPair ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = __shfl_sync(0xffffffffu, (smem_u32(smem_raw) + 1023u) & ~1023u, 0);
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int num_stages = args.num_stages;
  const uint32_t ring_bytes = static_cast<uint32_t>(num_stages) * kStageBytes;
  const uint32_t staging_base = smem_base + ring_bytes;
  const uint32_t bias_off = ring_bytes + kEpiWarps * kStagingDepth * kStagingBoxBytes;
  const uint32_t bar_off = bias_off + kEpiWarps * BN * 4;
  const uint32_t bar_base = smem_base + bar_off;
  const uint32_t full_bar0 = bar_base, empty_bar0 = bar_base + 8u * kMxMaxStages;
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * kMxMaxStages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * kMxMaxStages + 2 + b); };
  const uint32_t scale_bar0 = bar_base + 8u * (2 * kMxMaxStages + 4);
  constexpr uint32_t kNumBars = 3 * kMxMaxStages + 4;
  const uint32_t tmem_slot = bar_base + 8u * kNumBars;
  volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(smem_gen + bar_off + 8u * kNumBars);
  volatile uint32_t* abort_p = tmem_slot_p + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(full_bar0 + 8u * s, 1);
      mbar_init(empty_bar0 + 8u * s, 1);
      mbar_init(scale_bar0 + 8u * s, 2);   // a commit per warp that copies scales
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), (kPair ? 8 : 4) * kEpiGroups / kAcc);   // the warps that drain it, in both CTAs of a pair
    }
    *abort_p = 0u;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_sa);
    prefetch_tmap(&tmap_sw);
    if constexpr (kStore == kMxStoreTma) prefetch_tmap(&tmap_out);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair<kTmemCols>(tmem_slot);
      tmem_relinquish_pair();
    } else {
      tmem_alloc<kTmemCols>(tmem_slot);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot_p, 0);
  griddep_launch_dependents();
  griddep_wait();

  const int tiles = args.num_m_tiles * args.num_n_tiles;
  const int k_iters = args.k_iters;
  // panels of `panel_width` column tiles, row by row inside a panel: see the convolution's general kernel
  auto tile_coords = [&](int tile, int& mt, int& nt) {
    const int panel = tile / args.panel_tiles;
    const int rem = tile - panel * args.panel_tiles;
    const int n0 = panel * args.panel_width;
    const int width = min(args.panel_width, args.num_n_tiles - n0);
    mt = rem / width;
    nt = n0 + rem - mt * width;
  };
  const uint32_t full_leader0 = kPair ? __shfl_sync(0xffffffffu, mapa_cluster(full_bar0, 0u), 0) : full_bar0;
  const uint32_t ring_end = smem_base + ring_bytes;

  if (warp == 0 || warp == kSecondProducer) {
    // ------------------------------------------------------------ TMA producers (uniform control flow, one lane issues)
    // A warp needs ~140 cycles to issue a copy, whatever its size, and a stage has four: warp 0 brings A and its scales in, the other
    // one W and its. Only warp 0 arms the stage's barrier; bytes may arrive on it before, its phase cannot end without that.
    const uint32_t issue = elect_one_lane();
    uint32_t stage_addr = smem_base, full_addr = full_bar0, empty_addr = empty_bar0, phase = 0;
    bool ok = true, stopped = false;
    int issued = 0;
    for (int tile = worker; ok && !stopped && tile < tiles; tile += num_workers) {
      int mt, nt;
      tile_coords(tile, mt, nt);
      const int a_row = mt * kTileM + static_cast<int>(cta_rank) * kBlockM;
      const int w_row = nt * BN + static_cast<int>(cta_rank * kBRows);
      const int sa_tile = a_row / kMxTileRows, sw_tile = nt * BN / kMxTileRows;
      for (int it = 0; it < k_iters; ++it) {
        if (issued == args.test_producer_stop) {   // test hook: go silent, leave normally
          stopped = true;
          break;
        }
        if (!mbar_wait_bounded_uniform(empty_addr, phase ^ 1u, abort_p, args.wait_limit)) {
          if (issue) report_error_status(args.status, abort_p, kErrProducerWait, static_cast<uint32_t>(it));
          ok = false;
          break;
        }
        const uint32_t full = full_leader0 + (full_addr - full_bar0);
        if (warp == 0) {
          if (leader) mbar_arrive_expect_tx_if(issue, full_addr, kPair ? 2u * kStageBytes : kStageBytes);
          if constexpr (kPair) {
            tma_load_2d_pair_if(issue, stage_addr, &tmap_a, full, it * kStageKBytes, a_row);
            tma_load_3d_pair_if(issue, stage_addr + kSaOff, &tmap_sa, full, 0, 2 * it, sa_tile);
          } else {
            tma_load_2d_if(issue, stage_addr, &tmap_a, full, it * kStageKBytes, a_row);
            tma_load_3d_if(issue, stage_addr + kSaOff, &tmap_sa, full, 0, 2 * it, sa_tile);
          }
        } else if constexpr (kPair) {
          tma_load_2d_pair_if(issue, stage_addr + kABytes, &tmap_w, full, it * kStageKBytes, w_row);
          tma_load_3d_pair_if(issue, stage_addr + kSbOff, &tmap_sw, full, 0, 2 * it, sw_tile);
        } else {
          tma_load_2d_if(issue, stage_addr + kABytes, &tmap_w, full, it * kStageKBytes, w_row);
          tma_load_3d_if(issue, stage_addr + kSbOff, &tmap_sw, full, 0, 2 * it, sw_tile);
        }
        ++issued;
        stage_addr += kStageBytes; full_addr += 8u; empty_addr += 8u;
        if (stage_addr == ring_end) { stage_addr = smem_base; full_addr = full_bar0; empty_addr = empty_bar0; phase ^= 1u; }
      }
    }
    // never leave with copies in flight into this CTA's shared memory
    if (ok) {
      const int pending = issued < num_stages ? issued : num_stages;
      if (issued < num_stages) { stage_addr = smem_base; empty_addr = empty_bar0; phase = 1u; }   // the oldest filled stage; its first release has parity 0
      for (int i = 0; i < pending; ++i) {
        if (!mbar_wait_bounded_uniform(empty_addr, phase ^ 1u, abort_p, args.wait_limit)) break;
        stage_addr += kStageBytes; empty_addr += 8u;
        if (stage_addr == ring_end) { stage_addr = smem_base; empty_addr = empty_bar0; phase ^= 1u; }
      }
    } else {
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { __nanosleep(1000); }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (uniform control flow, one lane issues)
    if (leader) {
      const uint32_t issue = elect_one_lane();
      // operands: 128-byte swizzled rows, 8 rows to 1024 bytes
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t idesc0 = args.idesc, idesc2 = args.idesc | (2u << 4) | (2u << 29);   // scale words' lower and upper halves
      constexpr uint32_t kStageUnits = kStageBytes >> 4;
      // The ring's state, moved by additions: this loop, not the tensor pipe, sets the pace of a stage (with a multiplication for
      // every address 455 cycles, of which the MMAs of 256 x 192 take 384).
      const uint32_t a_first = smem_base >> 4, ta_first = tmem_base + kAcc * BN;
      const uint32_t a_end = a_first + static_cast<uint32_t>(num_stages) * kStageUnits;
      uint32_t a = a_first, ta = ta_first, bar = 0, phase = 0;
      int local = 0;
      uint32_t sw_shifts = 0;
      bool ok = true;
      bool ready = false;             // pairs: this stage's scales are known to be in place; else: the next stage's bytes are
      bool scales_issued = false;     // not pairs: this stage's scales are on their way to tensor memory
      // not pairs: the copies of a stage's scales. They run in order with this warp's MMAs, so no wait lies between
      auto copy_scales = [&](uint32_t stage_a, uint32_t dst) {
        constexpr uint32_t kScaleDescHi = (128u >> 4) | (1u << 14);   // 32 rows of 16 bytes, 8 rows to 128 bytes, not swizzled
        const uint32_t src = stage_a + (kSaOff >> 4);
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
          tmem_cp_32x128b_if<kPair>(issue, dst + 4u * k, src + k * (kMxTileBytes >> 4), kScaleDescHi);
#pragma unroll
          for (uint32_t r = 0; r < kBTiles; ++r)
            tmem_cp_32x128b_if<kPair>(issue, dst + 8u + 4u * (k * kBTiles + r), src + (2u + 2u * r + k) * (kMxTileBytes >> 4),
                                      kScaleDescHi);
        }
      };
      for (int tile = worker; ok && tile < tiles; tile += num_workers, ++local) {
        const int buf = kAcc == 2 ? local & 1 : 0;
        const uint32_t use = static_cast<uint32_t>(kAcc == 2 ? local >> 1 : local);
        if (!mbar_wait_bounded_uniform(tempty_bar(buf), (use & 1u) ^ 1u, abort_p, args.wait_limit)) {
          if (issue) report_error_status(args.status, abort_p, kErrMmaWaitTmem, static_cast<uint32_t>(local));
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sw_shift = 0;        // the tile may start inside a tile of scales
        if constexpr (BN % kMxTileRows != 0) {
          if ((local & 31) == 0) {    // a lane each for the next 32 tiles: the divisions would hold every tile up
            int mt, nt;
            tile_coords(min(tile + lane * num_workers, tiles - 1), mt, nt);
            sw_shifts = static_cast<uint32_t>(nt * BN % kMxTileRows) / 32u;
          }
          sw_shift = __shfl_sync(0xffffffffu, sw_shifts, local & 31);
        }
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(buf) * BN;
        for (int it = 0; it < k_iters; ++it) {
          uint32_t next_a = a + kStageUnits, next_ta = ta + kScaleCols, next_bar = bar + 8u, next_phase = phase;
          if (next_a == a_end) { next_a = a_first; next_ta = ta_first; next_bar = 0; next_phase ^= 1u; }
          uint32_t probe_bar = scale_bar0 + next_bar, probe_phase = next_phase;
          if constexpr (kPair) {
            if (!ready && !mbar_wait_bounded_uniform(scale_bar0 + bar, phase, abort_p, args.wait_limit)) {
              if (issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(it));
              ok = false;
              break;
            }
            tc_fence_after();
          } else {
            if (!scales_issued) {
              if (!mbar_wait_bounded_uniform(full_bar0 + bar, phase, abort_p, args.wait_limit)) {
                if (issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(it));
                ok = false;
                break;
              }
              tc_fence_after();
              copy_scales(a, ta);
            }
            // the next stage's scales go ahead of this stage's MMAs where its bytes are known to have landed: copies right in
            // front of the MMAs that read them hold the tensor pipe up. (Behind the last step there is no such stage: nobody
            // loads it, so the phase that the probe asks for does not end.)
            scales_issued = ready;
            if (scales_issued) {
              tc_fence_after();
              copy_scales(next_a, next_ta);
            }
            probe_bar = full_bar0 + next_bar + 8u;
            if (next_a + kStageUnits == a_end) { probe_bar = full_bar0; probe_phase ^= 1u; }
          }
          const uint32_t b = a + (kABytes >> 4), tb = ta + 8u + sw_shift;
          const bool landed = mx_mma_stage4_probe<kPair>(d_tmem, a, b, kDescHi, idesc0, idesc2, ta, ta + 4u, tb, tb + 4u * kBTiles,
                                                         empty_bar0 + bar, probe_bar, probe_phase, it != 0 ? 1u : 0u, issue);
          a = next_a; ta = next_ta; bar = next_bar; phase = next_phase;
          ready = __all_sync(0xffffffffu, landed);
        }
        if (ok && issue) {
          if constexpr (kPair) mma_commit_pair(tfull_bar(buf));
          else mma_commit(tfull_bar(buf));
        }
        __syncwarp();
      }
    }
  } else if (warp >= kScaleWarp) {
    // ------------------------------------------------------------ scales: shared memory -> tensor memory (uniform, one lane issues)
    // Warps of their own, each half of a stage's 256 columns: a copy takes ~50 cycles to issue, and with all of them in front of
    // the MMAs in one warp a stage took 830 cycles against 520 without them. These wait for the stage's bytes, the MMA warp for
    // the commits behind these copies. 8192^3: 279 us, 216 with one such warp, 213 with two.
    if (leader) {
      const uint32_t issue = elect_one_lane();
      constexpr uint32_t kScaleDescHi = (128u >> 4) | (1u << 14);   // 32 rows of 16 bytes, 8 rows to 128 bytes, not swizzled
      const uint32_t k = static_cast<uint32_t>(warp - kScaleWarp);
      const uint32_t src0 = (smem_base + kSaOff + k * kMxTileBytes) >> 4, dst0 = tmem_base + kAcc * BN;
      uint32_t src = src0, dst = dst0;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < tiles; tile += num_workers) {
        for (int it = 0; it < k_iters; ++it) {
          if (!mbar_wait_bounded_uniform(full_bar0 + 8u * stage, phase, abort_p, args.wait_limit)) {
            if (issue) report_error_status(args.status, abort_p, kErrMmaWaitFull, static_cast<uint32_t>(it));
            ok = false;
            break;
          }
          tc_fence_after();
          // [tile of rows][k tile] in shared memory -> [k tile][tile of rows] in tensor memory
          tmem_cp_32x128b_if<kPair>(issue, dst + 4u * k, src, kScaleDescHi);
#pragma unroll
          for (uint32_t r = 0; r < kBTiles; ++r)
            tmem_cp_32x128b_if<kPair>(issue, dst + 8u + 4u * (k * kBTiles + r), src + (2u + 2u * r) * (kMxTileBytes >> 4),
                                      kScaleDescHi);
          tcgen05_commit_if<kPair>(issue, scale_bar0 + 8u * stage);
          src += kStageBytes >> 4;
          dst += kScaleCols;
          if (++stage == num_stages) {
            stage = 0;
            phase ^= 1u;
            src = src0;
            dst = dst0;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: groups of four warps, a row a lane
    // With two accumulators, half of the groups take every second tile, and all of them the last one, which nothing overlaps; with
    // one accumulator all take every tile. Groups that share a tile take alternate groups of columns.
    const int ew = warp - 2, egroup = ew >> 2, quarter = warp & 3;
    constexpr int kShare = kEpiGroups / kAcc;
    constexpr int kGroupCols = kStore == kMxStoreMx ? 32 : 128 / static_cast<int>(sizeof(OutT));
    constexpr int kGroups = BN / kGroupCols;
    constexpr int kLdPerGroup = kGroupCols / 32;
    constexpr int kVec = 16 / sizeof(OutT);
    constexpr int kChunksPerLd = 32 / kVec;
    float* bias_w = reinterpret_cast<float*>(smem_gen + bias_off) + ew * BN;
    const uint32_t bias_s = smem_base + bias_off + static_cast<uint32_t>(ew * BN) * 4u;
    const uint32_t stg0 = staging_base + static_cast<uint32_t>(ew * kStagingDepth) * kStagingBoxBytes;
    const uint32_t lane_row_off = static_cast<uint32_t>(lane) * 128u, lane_xor = static_cast<uint32_t>(lane) & 7u;
    const OutT* res = static_cast<const OutT*>(args.residual);
    const int my_tiles = worker < tiles ? (tiles - worker + num_workers - 1) / num_workers : 0;
    uint32_t box = 0;
    // The bias of the tile after this one is on its way to registers while this one is waited for and finished (12544 x 4096 x 1024
    // bf16 30.4 us; 34.7 where each was loaded as its tile began). Tiles of 256 columns, for long K, have no registers for that.
    int bias_tile = -1, ahead_tile = -1;
    float ahead[BN / 32];
    auto load_bias = [&](int nt) {
      ahead_tile = nt;
#pragma unroll
      for (int j = 0; j < BN / 32; ++j) {
        const int n = nt * BN + j * 32 + lane;
        ahead[j] = 0.0f;
        if (args.bias != nullptr && n < args.N)
          ahead[j] = args.bias_is_f32 ? ld_global_f32(static_cast<const float*>(args.bias) + n)
                                      : OutTraits<OutT>::to_f(static_cast<const OutT*>(args.bias)[n]);
      }
    };
    auto next_tile = [&](int local) {
      ++local;
      if (kAcc == 2 && local < my_tiles - 1 && (local & 1) != egroup / kShare) ++local;
      return local;
    };
    bool ok = true;
    int local = next_tile(-1), mt = 0, nt = 0, local_next, mt_next = 0, nt_next = 0;
    if (local < my_tiles) tile_coords(worker + local * num_workers, mt, nt);
    for (; ok && local < my_tiles; local = local_next, mt = mt_next, nt = nt_next) {
      const bool last = kAcc == 2 && local == my_tiles - 1;
      local_next = next_tile(local);
      const int g_first = last ? egroup : egroup % kShare, g_step = last ? kEpiGroups : kShare;
      const int buf = kAcc == 2 ? local & 1 : 0;
      const uint32_t use = static_cast<uint32_t>(kAcc == 2 ? local >> 1 : local);
      const int n_base = nt * BN;
      const int m_row0 = mt * kTileM + static_cast<int>(cta_rank) * kBlockM + quarter * 32;
      const int m = m_row0 + lane;
      const bool row_ok = m < args.M;
      // the residual of the first groups of columns, one a box, while the accumulator is being computed
      int res_ahead = g_first;                     // the first group whose residual is not in its box
      if (kStore != kMxStoreMx && res != nullptr) {
        if (kStore == kMxStoreTma && lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        for (int d = 0; d < kStagingDepth && res_ahead < kGroups && n_base + res_ahead * kGroupCols < args.N; ++d) {
          const int n0 = n_base + res_ahead * kGroupCols;
          mx_fetch_rows<OutT>(args.res_vec, stg0 + (kStagingDepth == 2 ? box ^ (d & 1u) : 0u) * kStagingBoxBytes,
                              res, res + m_row0 * args.res_stride + n0, args.res_stride, args.M - m_row0, args.N - n0, lane);
          res_ahead += g_step;
        }
      }
      if (bias_tile < 0 || (args.bias != nullptr && nt != bias_tile)) {
        if (nt != ahead_tile) load_bias(nt);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < BN / 32; ++j) bias_w[j * 32 + lane] = ahead[j];
        __syncwarp();
        bias_tile = nt;
      }
      if (local_next < my_tiles) {
        tile_coords(worker + local_next * num_workers, mt_next, nt_next);
        if (BN < 256 && args.bias != nullptr && nt_next != bias_tile) load_bias(nt_next);
      }
      const bool ready = mbar_wait_bounded(tfull_bar(buf), use & 1u, abort_p, 2 * args.wait_limit);
      if (!__all_sync(0xffffffffu, ready)) {
        if (lane == 0) report_error_status(args.status, abort_p, kErrEpilogueWait, static_cast<uint32_t>(local));
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t taddr0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(buf) * BN;
#pragma unroll 1
      for (int g = g_first; g < kGroups; g += g_step) {
        const int n0 = n_base + g * kGroupCols;
        const bool live = n0 < args.N;
        uint32_t v[kLdPerGroup][32];
#pragma unroll
        for (int h = 0; h < kLdPerGroup; ++h) tmem_ld_32x32(taddr0 + g * kGroupCols + h * 32, v[h]);
        tmem_ld_wait();
        if (!last && g + kShare >= kGroups) {        // (nobody waits for the buffer of the last tile)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (kPair) mbar_arrive_cluster_relaxed(mapa_cluster(tempty_bar(buf), 0u));
            else mbar_arrive(tempty_bar(buf));
          }
        }
        if (!live) continue;
        const uint32_t stg = stg0 + box * kStagingBoxBytes;
        if constexpr (kStore == kMxStoreTma) {
          if (lane == 0) bulk_wait_group_read<kStagingDepth - 1>();   // this box's last store has been read out
          __syncwarp();
        }
        if constexpr (kStore != kMxStoreMx) {
          if (res != nullptr) {
            if (g >= res_ahead)
              mx_fetch_rows<OutT>(args.res_vec, stg, res, res + m_row0 * args.res_stride + n0, args.res_stride, args.M - m_row0,
                                  args.N - n0, lane);
            cp_async_wait_all();
            __syncwarp();                              // rows come from other lanes than the ones that add them
          }
        }
        uint4 packed[8];
        uint32_t scale_bytes = 0;
#pragma unroll
        for (int h = 0; h < kLdPerGroup; ++h) {
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[h][j]);
#pragma unroll
          for (int j4 = 0; j4 < 8; ++j4) {
            const float4 b4 = ld_shared_f4(bias_s + static_cast<uint32_t>(g * kGroupCols + h * 32 + j4 * 4) * 4u);
            add2(f[j4 * 4 + 0], f[j4 * 4 + 1], b4.x, b4.y);
            add2(f[j4 * 4 + 2], f[j4 * 4 + 3], b4.z, b4.w);
          }
          // columns past N: their scales are whatever lies behind the last row of W, and may not reach their neighbours' results
          if (n0 + h * 32 + 32 > args.N) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (n0 + h * 32 + j >= args.N) f[j] = 0.0f;
          }
          if constexpr (kStore == kMxStoreMx) {
            mx_act32<true>(f, args.act);
            uint32_t byte;
            packed[h] = mx_quantize32(f, byte);
            scale_bytes = byte;
          } else {
            if (res != nullptr) {
#pragma unroll
              for (int c = 0; c < kChunksPerLd; ++c) {
                const uint32_t cc = static_cast<uint32_t>(h * kChunksPerLd + c);
                add16<OutT>(f + c * kVec, ld_shared_v4(stg + lane_row_off + ((cc ^ lane_xor) << 4)));
              }
            }
            if (sizeof(OutT) == 2 && args.act == kActRelu) {        // in the rounding, which keeps NaN
              finish32<OutT, true>(f, nullptr, false, packed + h * kChunksPerLd);
            } else {
              mx_act32<sizeof(OutT) == 2>(f, args.act);
              finish32<OutT, false>(f, nullptr, false, packed + h * kChunksPerLd);
            }
          }
        }
        if constexpr (kStore == kMxStoreMx) {
          // a block of this lane's row; behind the last one, the rest of its word of scales is 0
          const int blk = n0 / kMxBlock;
          if (row_ok) {
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(args.out) + static_cast<long long>(m) * (16LL * args.out_blocks) + 16LL * blk) =
                packed[0];
            uint8_t* sw = args.out_scales + mx_scale_word(m, blk >> 2, args.out_k_tiles);
            sw[blk & 3] = static_cast<uint8_t>(scale_bytes);
            if (blk + 1 == args.out_blocks)
              for (int b = (blk & 3) + 1; b < 4; ++b) sw[b] = 0;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            st_shared_v4(stg + lane_row_off + ((static_cast<uint32_t>(c) ^ lane_xor) << 4), packed[c]);
          if constexpr (kStore == kMxStoreTma) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_out, stg, n0, m_row0);
              bulk_commit_group();
            }
            if constexpr (kStagingDepth == 2) box ^= 1u;
          } else {
            mx_store_rows<OutT>(args.out_vec, stg, static_cast<OutT*>(args.out) + m_row0 * args.out_stride + n0, args.out_stride,
                                args.M - m_row0, args.N - n0, lane);
            if constexpr (kStagingDepth == 2) box ^= 1u;
          }
        }
      }
    }
    if (kStore == kMxStoreTma && lane == 0) bulk_wait_group0();
  }

  tc_fence_before();
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair<kTmemCols>(tmem_base);
    else tmem_dealloc<kTmemCols>(tmem_base);
  }
}

}  // namespace tb200
