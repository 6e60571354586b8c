// The norm in front of a block and the join behind it, one pass over the rows:
//   join:  r = residual_scale * x + gate * stage(h)
//   norm:  y = stage(r), in the storage type or in the 4-bit format of mx_format.cuh
// where stage(v) = (norm(v) * weight + bias) * (1 + scale) + shift, and norm(v) = v / sqrt(mean(v^2) + eps) (rms),
// (v - mean) / sqrt(mean((v - mean)^2) + eps) (layer) or v (none). A call does either or both; the norm behind a join reads r as it
// is stored, so that both in one call give the bits of two calls where all their rows allow the same accesses (16 bytes or not). A
// row that is summed in the other form's order differs by fp32's rounding.
//
// Bound by memory: a row is read once into registers and everything is computed from there, in fp32. The second moment is taken
// about the mean, in a pass of its own over the registers -- as mean(v^2) - mean^2 a row far from zero would lose it.
//
// A row belongs to a group of 32 to 512 threads with up to 32 columns each: what a thread does per row and not per column --
// sums across threads, addresses, the loop -- is as many instructions as eight columns take (12544 x 1024 modulated: with eight
// columns a thread 16.0 us, sixteen 12.6, 32 11.4, captured, the same input over and over; 13.9 a call where the inputs change). A CTA
// walks consecutive rows. The vectors per channel, as many bytes as
// several rows, come to v -> v * a + b, which is kept in shared memory until the group of rows changes (up to 8192 columns).
// Meanwhile rows are on their way: each thread copies its own columns to a ring in shared memory, several rows ahead, and needs
// no barrier for them.
#pragma once
#include "mx_format.cuh"

namespace tb200 {

enum : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum : int { kNextNone = 0, kNextRows = 1, kNextMx = 2 };

// A vector of a value per channel, or one of these per group of rows. f32: in fp32, else in the rows' type.
struct NormVector {
  const void* ptr;
  long long group_stride;   // elements; 0 where there is one for all rows
  int f32;
  int vec;                  // eight columns from a multiple of eight on are 16-byte aligned
};
struct NormStage {
  int kind;
  float eps;
  NormVector weight, bias, scale, shift;
};
struct BlockNormArgs {
  const void* h;            // join: what the block computed
  const void* x;            // join: the residual stream; else the rows to be normed
  void* r;                  // join: its result
  void* y;                  // the norm's result
  uint8_t* codes;           // the same in 4 bits
  uint8_t* scales;
  long long h_stride, x_stride, r_stride, y_stride;   // rows, in elements
  int M, rows_per_group;
  int C, blocks, k_tiles;
  float residual_scale;
  NormVector gate;
  NormStage join, norm;
};

// How a thread's eight columns of a vector lie and are moved: consecutive ones in 16-byte accesses; consecutive ones one by one;
// or, where nothing needs neighbours, kThreads apart, so that a warp's accesses are consecutive.
enum : int { kRowsVec = 0, kRowsSingle = 1, kRowsSpread = 2 };

template <typename T, int kMode, int kThreads>
struct RowSlice {
  static constexpr int kBytes = 8 * sizeof(T);
  __device__ __forceinline__ static int col(int i, int t, int j) {
    return kMode == kRowsSpread ? (i * 8 + j) * kThreads + t : (i * kThreads + t) * 8 + j;
  }
  __device__ __forceinline__ static void load(const T* p, int i, int t, int C, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col(i, t, j) < C ? OutTraits<T>::to_f(p[col(i, t, j)]) : 0.0f;
  }
  // kRowsVec: the same by way of shared memory. Columns past C are never copied: their places hold zeros from the start.
  __device__ __forceinline__ static void copy(uint32_t smem, const T* p, int i, int t, int C, bool live) {
    if (live && col(i, t, 0) < C) {
#pragma unroll
      for (int q = 0; q < kBytes / 16; ++q) ptx::cp_async_16(smem + 16 * q, reinterpret_cast<const uint4*>(p + col(i, t, 0)) + q);
    }
  }
  __device__ __forceinline__ static void copied(uint32_t smem, float (&v)[8]) {
    __align__(16) uint4 raw[kBytes / 16];
#pragma unroll
    for (int q = 0; q < kBytes / 16; ++q) raw[q] = ptx::ld_shared_v4(smem + 16 * q);
    load8<T>(reinterpret_cast<const T*>(raw), v);
  }
  __device__ __forceinline__ static void zero(uint32_t smem) {
#pragma unroll
    for (int q = 0; q < kBytes / 16; ++q) ptx::st_shared_v4(smem + 16 * q, make_uint4(0u, 0u, 0u, 0u));
  }
  __device__ __forceinline__ static void store(T* p, int i, int t, int C, const float (&v)[8]) {
    if constexpr (kMode == kRowsVec) {
      if (col(i, t, 0) < C) store8<T>(p + col(i, t, 0), v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col(i, t, j) < C) p[col(i, t, j)] = OutTraits<T>::from_f(v[j]);
    }
  }
};

// Eight columns of a vector per channel (undefined past C), or `missing` where there is none.
template <typename T, int kMode, int kThreads>
__device__ __forceinline__ void norm_vector8(const NormVector& p, float missing, int group, int i, int t, int C, float (&v)[8]) {
  using Slice = RowSlice<T, kMode, kThreads>;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = missing;
  if (p.ptr == nullptr) return;
  const long long at = group * p.group_stride;
  if (kMode == kRowsVec && p.vec) {
    if (Slice::col(i, t, 0) < C) {
      if (p.f32) load8<float>(static_cast<const float*>(p.ptr) + at + Slice::col(i, t, 0), v);
      else load8<T>(static_cast<const T*>(p.ptr) + at + Slice::col(i, t, 0), v);
    }
  } else if (p.f32) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (Slice::col(i, t, j) < C) v[j] = static_cast<const float*>(p.ptr)[at + Slice::col(i, t, j)];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (Slice::col(i, t, j) < C) v[j] = OutTraits<T>::to_f(static_cast<const T*>(p.ptr)[at + Slice::col(i, t, j)]);
  }
}

// What a stage's vectors, and a join's gate, come to: v -> v * a + b.
template <typename T, int kMode, int kThreads>
__device__ __forceinline__ void norm_affine8(const NormStage& s, const NormVector* gate, int group, int i, int t, int C,
                                             float (&a)[8], float (&b)[8]) {
  float scale[8], shift[8], g[8];
  norm_vector8<T, kMode, kThreads>(s.weight, 1.0f, 0, i, t, C, a);
  norm_vector8<T, kMode, kThreads>(s.bias, 0.0f, 0, i, t, C, b);
  norm_vector8<T, kMode, kThreads>(s.scale, 0.0f, group, i, t, C, scale);
  norm_vector8<T, kMode, kThreads>(s.shift, 0.0f, group, i, t, C, shift);
  if (gate != nullptr) norm_vector8<T, kMode, kThreads>(*gate, 1.0f, group, i, t, C, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a[j] = fmaf(a[j], scale[j], a[j]);
    b[j] = fmaf(b[j], scale[j], b[j]) + shift[j];
    if (gate != nullptr) {
      a[j] *= g[j];
      b[j] *= g[j];
    }
  }
}
__device__ __forceinline__ bool has_shift(const NormStage& s) { return s.bias.ptr != nullptr || s.shift.ptr != nullptr; }

// A CTA's rows are walked by groups of kThreads threads. A join's CTA is as large as an SM holds where rows are short: with 256
// threads each, copies of the vectors took shared memory that rows on their way can use (65536 x 256 bf16 and next norm 24.5 ->
// 20.9 us; of 1001 columns, 333 rows, it would cost, 3.7 -> 4.8, of 4096, 91 -> 100).
__host__ __device__ constexpr int norm_block_threads(int row_threads, int vecs, bool join) {
  return join && row_threads == 32 && vecs <= 2 ? 768 : (row_threads < 256 ? 256 : row_threads);
}

// A barrier of the threads of a row.
template <int kThreads, int kBlock>
__device__ __forceinline__ void row_barrier(int warp) {
  if constexpr (kThreads == 32) __syncwarp();
  else if constexpr (kThreads == kBlock) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / (kThreads / 32)), "n"(kThreads) : "memory");
}

// The sum over the threads of a row, in every one of them, always in the same order. `slot` alternates between two buffers: the
// barrier of one sum is behind every read of the sum before it.
template <int kThreads, int kBlock>
__device__ __forceinline__ float row_sum(float v, float* smem, uint32_t& slot, int lane, int warp) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    float* s = smem + slot * 32;
    slot ^= 1u;
    if (lane == 0) s[warp] = v;
    row_barrier<kThreads, kBlock>(warp);
    s += warp / kWarps * kWarps;                 // the row's warps
    if constexpr (kWarps == 2) {
      v = s[0] + s[1];
    } else {
      v = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps / 4; ++i) {
        const float4 q = reinterpret_cast<const float4*>(s)[i];
        v += (q.x + q.y) + (q.z + q.w);
      }
    }
  }
  return v;
}

// v, the row with zeros past column C, becomes norm(v), zeros where they were.
template <int kMode, int kThreads, int kVecs, int kBlock>
__device__ __forceinline__ void norm_row(const NormStage& s, float (&v)[kVecs][8], int C, float inv_C, int t, float* smem,
                                         uint32_t& slot, int lane, int warp) {
  using Slice = RowSlice<float, kMode, kThreads>;
  if (s.kind == kNormNone) return;
  if (s.kind == kNormLayer) {
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 8; j += 2) add2(a, b, v[i][j], v[i][j + 1]);
    // divided, not multiplied by 1 / C: the mean of a constant row is its constant then, where the sums are exact
    const float mean = row_sum<kThreads, kBlock>(a + b, smem, slot, lane, warp) / static_cast<float>(C);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float m0 = Slice::col(i, t, kMode == kRowsVec ? 0 : j) < C ? mean : 0.0f;
        const float m1 = Slice::col(i, t, kMode == kRowsVec ? 0 : j + 1) < C ? mean : 0.0f;
        add2(v[i][j], v[i][j + 1], -m0, -m1);
      }
  }
  float a = 0.0f, b = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float x = v[i][j], y = v[i][j + 1];
      fma2(x, y, x, y, a, b);
      a = x;
      b = y;
    }
  const float inv = rsqrtf(fmaf(row_sum<kThreads, kBlock>(a + b, smem, slot, lane, warp), inv_C, s.eps));
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) mul2(v[i][j], v[i][j + 1], inv, inv);
}

// The CTA's copy of a stage's a, then its b: slice (i, t)'s eight values as two halves of four, the first halves of all slices in
// front, so that neighbouring threads' accesses are neighbours.
template <int kSlices>
__device__ __forceinline__ void norm_keep(float* kept, int slice, const float (&a)[8], const float (&b)[8]) {
  float4* k = reinterpret_cast<float4*>(kept) + slice;
  k[0] = make_float4(a[0], a[1], a[2], a[3]);
  k[kSlices] = make_float4(a[4], a[5], a[6], a[7]);
  k[2 * kSlices] = make_float4(b[0], b[1], b[2], b[3]);
  k[3 * kSlices] = make_float4(b[4], b[5], b[6], b[7]);
}

// v -> v * a + b, from the CTA's copy (kKeep) or from the vectors.
template <typename T, int kMode, int kThreads, int kVecs, bool kKeep>
__device__ __forceinline__ void norm_apply8(const NormStage& s, const NormVector* gate, const float* kept, int group, bool shift,
                                            int i, int t, int C, float (&v)[8]) {
  constexpr int kSlices = kThreads * kVecs;
  float a[8], b[8];
  if constexpr (kKeep) {
    const float4* k = reinterpret_cast<const float4*>(kept) + (i * kThreads + t);
    *reinterpret_cast<float4*>(a) = k[0];
    *reinterpret_cast<float4*>(a + 4) = k[kSlices];
    if (shift) {
      *reinterpret_cast<float4*>(b) = k[2 * kSlices];
      *reinterpret_cast<float4*>(b + 4) = k[3 * kSlices];
    }
  } else {
    norm_affine8<T, kMode, kThreads>(s, gate, group, i, t, C, a, b);
  }
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    if (shift) fma2(v[j], v[j + 1], a[j], a[j + 1], b[j], b[j + 1]);
    else mul2(v[j], v[j + 1], a[j], a[j + 1]);
  }
}

// The shape of a launch: shared memory is the CTA's copy of up to two stages' vectors, then (kRowsVec) the ring of rows.
__host__ __device__ constexpr bool norm_keeps(int threads, int vecs) { return threads * vecs * 8 <= 8192; }
__host__ __device__ constexpr int norm_kept_bytes(int threads, int vecs, bool join, int next) {
  return norm_keeps(threads, vecs) ? threads * vecs * 8 * 2 * 4 * ((join ? 1 : 0) + (next != kNextNone ? 1 : 0)) : 0;
}
__host__ __device__ constexpr int norm_row_bytes(int threads, int vecs, bool join, int es) {
  return norm_block_threads(threads, vecs, join) * vecs * 8 * es * (join ? 2 : 1);
}
// CTAs an SM is to hold: 1024 threads of 64 registers; joins 768 of 80 or 512 of 128. More than sixteen columns a thread: 512, in fp32
// 768 (12544 x 768 fp32 16.9 -> 15.4 us; bf16, 1024 columns, quantised 14.6 -> 15.3).
__host__ __device__ constexpr int norm_blocks_per_sm(int threads, int vecs, bool join, int es) {
  return join && threads == 32 && vecs <= 2 ? 1 : (join ? 512 : (vecs <= 2 ? 1024 : (es == 4 ? 768 : 512))) / norm_block_threads(threads, vecs, join);
}
// Rows ahead: what the CTA's share of 190 KB of shared memory holds, four at most.
__host__ __device__ constexpr int norm_depth(int threads, int vecs, bool join, int next, int es) {
  const int n = (190 * 1024 / norm_blocks_per_sm(threads, vecs, join, es) - norm_kept_bytes(threads, vecs, join, next)) /
                norm_row_bytes(threads, vecs, join, es);
  return n > 4 ? 4 : (n < 1 ? 1 : n);
}
// kRowsSingle, joins: the join is done with the columns spread, as where its rows are not quantised, so that it gives the same bits
// whatever follows it; its result changes hands through shared memory, a row of fp32 for every row in hand.
__host__ __device__ constexpr int norm_join_mode(int mode) { return mode == kRowsSingle ? kRowsSpread : mode; }
__host__ __device__ constexpr int norm_smem_bytes(int threads, int vecs, int mode, bool join, int next, int es) {
  return norm_kept_bytes(threads, vecs, join, next) +
         (mode == kRowsVec ? norm_depth(threads, vecs, join, next, es) * norm_row_bytes(threads, vecs, join, es)
                           : (mode == kRowsSingle && join ? norm_block_threads(threads, vecs, join) * vecs * 8 * 4 : 0));
}

template <typename T, int kThreads, int kVecs, int kMode, bool kJoin, int kNext>
__global__ void __launch_bounds__(norm_block_threads(kThreads, kVecs, kJoin), norm_blocks_per_sm(kThreads, kVecs, kJoin, sizeof(T)))
block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
  static_assert(!(kMode == kRowsSpread && kNext == kNextMx), "a block of the format is four neighbouring threads' columns");
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ __align__(16) float sums[64];
  using Slice = RowSlice<T, kMode, kThreads>;
  constexpr int kJoinMode = norm_join_mode(kMode);
  using JoinSlice = RowSlice<T, kJoin ? kJoinMode : kMode, kThreads>;
  constexpr int kBlock = norm_block_threads(kThreads, kVecs, kJoin);
  constexpr int kRows = kBlock / kThreads;                              // that a CTA has in hand at a time
  constexpr bool kKeep = norm_keeps(kThreads, kVecs);
  constexpr int kSlices = kThreads * kVecs;                             // of eight columns
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = static_cast<int>(threadIdx.x) % kThreads, sub = static_cast<int>(threadIdx.x) / kThreads;
  const int C = a.C;
  const float inv_C = 1.0f / static_cast<float>(C);
  const bool join_shift = kJoin && has_shift(a.join), norm_shift = has_shift(a.norm);
  float* kept_join = reinterpret_cast<float*>(dynamic);
  float* kept_norm = kept_join + (kJoin ? 16 * kSlices : 0);
  uint32_t slot = 0;

  // kRowsVec: ring slots [row][matrix][i][thread]
  constexpr int kDepth = norm_depth(kThreads, kVecs, kJoin, kNext, sizeof(T));
  constexpr uint32_t kRowBytes = norm_row_bytes(kThreads, kVecs, kJoin, sizeof(T));
  constexpr uint32_t kSliceBytes = kRowBytes / (kVecs * (kJoin ? 2 : 1));
  const uint32_t ring0 = ptx::smem_u32(dynamic) + norm_kept_bytes(kThreads, kVecs, kJoin, kNext) + threadIdx.x * Slice::kBytes;
  uint32_t ring_at = ring0;

  if constexpr (kMode == kRowsVec) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (Slice::col(i, t, 0) >= C)
#pragma unroll 1
        for (uint32_t at = ring0 + i * kSliceBytes; at < ring0 + kDepth * kRowBytes; at += kVecs * kSliceBytes) Slice::zero(at);
  }
  const int first = static_cast<int>(static_cast<long long>(blockIdx.x) * a.M / gridDim.x);
  const int last = static_cast<int>((static_cast<long long>(blockIdx.x) + 1) * a.M / gridDim.x);
  for (int seg = first; seg < last;) {                                  // rows of one group
    const int group = a.rows_per_group > 0 ? seg / a.rows_per_group : 0;
    const int seg_end = a.rows_per_group > 0 ? min(last, (group + 1) * a.rows_per_group) : last;
    int row = seg + sub;
    seg = seg_end;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* h = static_cast<const T*>(a.h) + (kJoin ? row * a.h_stride : 0);
    const long long x_step = kRows * a.x_stride, h_step = kRows * a.h_stride;
    int ahead = row;                                                    // the next row to be asked for, where x and h point
    auto request = [&]() {                                              // into the slot that has been read last
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        Slice::copy(ring_at + i * kSliceBytes, x, i, t, C, ahead < seg_end);
        if constexpr (kJoin) Slice::copy(ring_at + (kVecs + i) * kSliceBytes, h, i, t, C, ahead < seg_end);
      }
      ptx::cp_async_commit();
      ring_at = ring_at == ring0 + (kDepth - 1) * kRowBytes ? ring0 : ring_at + kRowBytes;
      x += x_step;
      if constexpr (kJoin) h += h_step;
      ahead += kRows;
    };
    if constexpr (kMode == kRowsVec) {
#pragma unroll 1
      for (int d = 0; d < kDepth; ++d) request();
    }
    if constexpr (kKeep) {
      // with one row in hand a thread reads only what it has written
      if constexpr (kRows > 1) __syncthreads();                         // the segment before has read its copy
#pragma unroll
      for (int n = 0; n < (kSlices + kBlock - 1) / kBlock; ++n) {
        const int slice = n * kBlock + static_cast<int>(threadIdx.x);
        if (kSlices % kBlock == 0 || slice < kSlices) {
          float p[8], q[8];
          if constexpr (kJoin) {
            norm_affine8<T, kJoinMode, kThreads>(a.join, &a.gate, group, slice / kThreads, slice % kThreads, C, p, q);
            norm_keep<kSlices>(kept_join, slice, p, q);
          }
          if constexpr (kNext != kNextNone) {
            norm_affine8<T, kMode, kThreads>(a.norm, nullptr, group, slice / kThreads, slice % kThreads, C, p, q);
            norm_keep<kSlices>(kept_norm, slice, p, q);
          }
        }
      }
      if constexpr (kRows > 1) __syncthreads();
    }
    T* r = static_cast<T*>(a.r) + row * a.r_stride;
    T* y = static_cast<T*>(a.y) + row * a.y_stride;
    for (; row < seg_end; row += kRows) {
      float v[kVecs][8];
      float xv[kVecs][8];
      if constexpr (kMode == kRowsVec) ptx::cp_async_wait<kDepth - 1>();
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        float(&xd)[8] = kJoin ? xv[i] : v[i];
        if constexpr (kMode == kRowsVec) {
          Slice::copied(ring_at + i * kSliceBytes, xd);
          if constexpr (kJoin) Slice::copied(ring_at + (kVecs + i) * kSliceBytes, v[i]);
        } else {
          JoinSlice::load(x, i, t, C, xd);
          if constexpr (kJoin) JoinSlice::load(h, i, t, C, v[i]);
        }
      }
      if constexpr (kMode == kRowsVec) {
        request();
      } else {
        x += x_step;
        if constexpr (kJoin) h += h_step;
      }
      if constexpr (kJoin) {
        norm_row<kJoinMode, kThreads, kVecs, kBlock>(a.join, v, C, inv_C, t, sums, slot, lane, warp);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          norm_apply8<T, kJoinMode, kThreads, kVecs, kKeep>(a.join, &a.gate, kept_join, group, join_shift, i, t, C, v[i]);
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            float p = xv[i][j], q = xv[i][j + 1];
            fma2(p, q, a.residual_scale, a.residual_scale, v[i][j], v[i][j + 1]);
            v[i][j] = p;
            v[i][j + 1] = q;
          }
          if constexpr (kMode == kRowsVec && sizeof(T) == 2) {         // rounded once, stored and read back from that
            uint4 w;
            w.x = pack2<T, false>(v[i][0], v[i][1]);
            w.y = pack2<T, false>(v[i][2], v[i][3]);
            w.z = pack2<T, false>(v[i][4], v[i][5]);
            w.w = pack2<T, false>(v[i][6], v[i][7]);
            if (JoinSlice::col(i, t, 0) < C) *reinterpret_cast<uint4*>(r + JoinSlice::col(i, t, 0)) = w;
            load8<T>(reinterpret_cast<const T*>(&w), v[i]);
          } else {
            JoinSlice::store(r, i, t, C, v[i]);
          }
          if constexpr (kNext != kNextNone && !(kMode == kRowsVec && sizeof(T) == 2)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[i][j] = OutTraits<T>::to_f(OutTraits<T>::from_f(v[i][j]));
              if (kMode != kRowsVec && JoinSlice::col(i, t, j) >= C) v[i][j] = 0.0f;    // kRowsVec: it is, a being 1 and b 0 there
            }
          }
        }
        r += kRows * a.r_stride;
        if constexpr (kJoinMode != kMode) {
          float* exchange = reinterpret_cast<float*>(dynamic + norm_kept_bytes(kThreads, kVecs, kJoin, kNext)) + sub * kSlices * 8;
#pragma unroll
          for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) exchange[JoinSlice::col(i, t, j)] = v[i][j];
          row_barrier<kThreads, kBlock>(warp);
#pragma unroll
          for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = exchange[Slice::col(i, t, j)];
          row_barrier<kThreads, kBlock>(warp);                                  // before the next row is written there
        }
      }
      if constexpr (kNext != kNextNone) {
        norm_row<kMode, kThreads, kVecs, kBlock>(a.norm, v, C, inv_C, t, sums, slot, lane, warp);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          norm_apply8<T, kMode, kThreads, kVecs, kKeep>(a.norm, nullptr, kept_norm, group, norm_shift, i, t, C, v[i]);
          if constexpr (kNext == kNextRows) {
            Slice::store(y, i, t, C, v[i]);
          } else {
            const int col = Slice::col(i, t, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (kMode != kRowsVec && col + j >= C) v[i][j] = 0.0f;
            uint32_t byte;
            const uint32_t codes = mx_quantize8(v[i], byte);            // the whole warp: blocks are shared by lanes
            if ((col >> 5) < a.blocks) *reinterpret_cast<uint32_t*>(a.codes + row * (16LL * a.blocks) + (col >> 1)) = codes;
            else if (kMode == kRowsVec) byte = 0u;                      // past the last block: 0 times the row's factor, which may be NaN
            if ((lane & 3) == 0 && (col >> 7) < a.k_tiles)
              a.scales[mx_scale_word(row, col >> 7, a.k_tiles) + ((col >> 5) & 3)] = static_cast<uint8_t>(byte);
          }
        }
        y += kRows * a.y_stride;
      }
    }
    if constexpr (kMode == kRowsVec) ptx::cp_async_wait<0>();
  }
}

}  // namespace tb200
