// The norm in front of a block and the join behind it, one pass over the rows:
//   join:  r = residual_scale * x + gate * stage(h)
//   norm:  y = stage(r), in the storage type or in the 4-bit format of mx_format.cuh
// where stage(v) = (norm(v) * weight + bias) * (1 + scale) + shift, and norm(v) = v / sqrt(mean(v^2) + eps) (rms),
// (v - mean) / sqrt(mean((v - mean)^2) + eps) (layer) or v (none). A call does either or both; the norm behind a join reads r as it
// is stored, so that both in one call give the bits of two calls.
//
// Bound by memory: a row is read once into registers and everything is computed from there, in fp32. The second moment is taken
// about the mean, in a pass of its own over the registers -- as mean(v^2) - mean^2 a row far from zero would lose it.
//
// A row belongs to a warp (up to 256 columns) or to a CTA whose threads hold eight columns each. The vectors per channel are as
// many bytes as several rows: a CTA walks consecutive rows and keeps what they come to, v -> v * a + b, in registers until the
// group of rows changes. It loads the next row before it works on this one.
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
  int vec;                  // 16-byte loads of eight columns are aligned
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
  long long M, rows_per_group;
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
  uint4 raw[sizeof(T) / 2];           // kRowsVec: as loaded, so that the load can be far ahead of its use
  float val[kMode == kRowsVec ? 1 : 8];
  __device__ __forceinline__ static int col(int i, int t, int j) {
    return kMode == kRowsSpread ? (i * 8 + j) * kThreads + t : (i * kThreads + t) * 8 + j;
  }
  __device__ __forceinline__ void load(const T* p, int i, int t, int C, bool live) {
    if constexpr (kMode == kRowsVec) {
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q)
        raw[q] = live && col(i, t, 0) < C ? reinterpret_cast<const uint4*>(p + col(i, t, 0))[q] : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) val[j] = live && col(i, t, j) < C ? OutTraits<T>::to_f(p[col(i, t, j)]) : 0.0f;
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (kMode == kRowsVec) {
      load8<T>(reinterpret_cast<const T*>(raw), v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = val[j];
    }
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

// Eight columns of a vector per channel (0 past C), or `missing` where there is none.
template <typename T, int kMode, int kThreads>
__device__ __forceinline__ void norm_vector8(const NormVector& p, float missing, long long group, int i, int t, int C, float (&v)[8]) {
  if (p.ptr == nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = missing;
    return;
  }
  const long long at = group * p.group_stride;
  using F = RowSlice<float, kMode, kThreads>;
  if constexpr (kMode == kRowsVec) {
    if (p.vec) {
      if (p.f32) {
        F s;
        s.load(static_cast<const float*>(p.ptr) + at, i, t, C, true);
        s.get(v);
      } else {
        RowSlice<T, kMode, kThreads> s;
        s.load(static_cast<const T*>(p.ptr) + at, i, t, C, true);
        s.get(v);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = F::col(i, t, j);
    v[j] = c >= C ? 0.0f : (p.f32 ? static_cast<const float*>(p.ptr)[at + c] : OutTraits<T>::to_f(static_cast<const T*>(p.ptr)[at + c]));
  }
}

// What a stage's vectors, and a join's gate, come to: v -> v * a + b.
template <typename T, int kMode, int kThreads>
__device__ __forceinline__ void affine8(const NormStage& s, const NormVector* gate, long long group, int i, int t, int C,
                                        float (&a)[8], float (&b)[8]) {
  float p[8];
  norm_vector8<T, kMode, kThreads>(s.weight, 1.0f, group, i, t, C, a);
  norm_vector8<T, kMode, kThreads>(s.bias, 0.0f, group, i, t, C, b);
  if (s.scale.ptr != nullptr) {
    norm_vector8<T, kMode, kThreads>(s.scale, 0.0f, group, i, t, C, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = fmaf(a[j], p[j], a[j]);
      b[j] = fmaf(b[j], p[j], b[j]);
    }
  }
  if (s.shift.ptr != nullptr) {
    norm_vector8<T, kMode, kThreads>(s.shift, 0.0f, group, i, t, C, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] += p[j];
  }
  if (gate != nullptr && gate->ptr != nullptr) {
    norm_vector8<T, kMode, kThreads>(*gate, 1.0f, group, i, t, C, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] *= p[j];
      b[j] *= p[j];
    }
  }
}

// The sum over the threads of a row, in every one of them, always in the same order. `slot` alternates between two buffers: the
// barrier of one sum is behind every read of the sum before it.
template <int kThreads>
__device__ __forceinline__ float row_sum(float v, float* smem, uint32_t& slot, int lane, int warp) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    float* s = smem + slot * 32;
    slot ^= 1u;
    if (lane == 0) s[warp] = v;
    __syncthreads();
    if constexpr (kWarps <= 8) {
      float4 q[kWarps / 4];
#pragma unroll
      for (int i = 0; i < kWarps / 4; ++i) q[i] = reinterpret_cast<const float4*>(s)[i];
      v = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps / 4; ++i) v += (q[i].x + q[i].y) + (q[i].z + q[i].w);
    } else {
      v = lane < kWarps ? s[lane] : 0.0f;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    }
  }
  return v;
}

// v, the row with zeros past column C, becomes norm(v); columns past C are undefined.
template <int kMode, int kThreads, int kVecs>
__device__ __forceinline__ void norm_row(const NormStage& s, float (&v)[kVecs][8], int C, int t, float* smem, uint32_t& slot,
                                         int lane, int warp) {
  if (s.kind == kNormNone) return;
  float mean = 0.0f;
  if (s.kind == kNormLayer) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[i][j];
    mean = row_sum<kThreads>(sum, smem, slot, lane, warp) / static_cast<float>(C);
  }
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] -= mean;
      if (RowSlice<float, kMode, kThreads>::col(i, t, j) < C) sq = fmaf(v[i][j], v[i][j], sq);
    }
  const float inv = rsqrtf(row_sum<kThreads>(sq, smem, slot, lane, warp) / static_cast<float>(C) + s.eps);
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] *= inv;
}

__host__ __device__ constexpr int norm_block_threads(int row_threads) { return row_threads == 32 ? 256 : row_threads; }
// CTAs an SM is to hold: 1024 threads of up to 64 registers, joins, which keep more, 768 of up to 80 (512 of 128 where a CTA is as many).
__host__ __device__ constexpr int norm_blocks_per_sm(int row_threads, bool join) {
  return row_threads == 1024 ? 1 : (join ? 768 : 1024) / norm_block_threads(row_threads);
}

template <typename T, int kThreads, int kVecs, int kMode, bool kJoin, int kNext>
__global__ void __launch_bounds__(norm_block_threads(kThreads), norm_blocks_per_sm(kThreads, kJoin))
block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
  static_assert(!(kMode == kRowsSpread && kNext == kNextMx), "a block of the format is four neighbouring threads' columns");
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  __shared__ __align__(16) float smem[64];
  using Slice = RowSlice<T, kMode, kThreads>;
  constexpr int kRows = norm_block_threads(kThreads) / kThreads;        // that a CTA has in hand at a time
  constexpr bool kKeep = kVecs == 1 && kThreads < 1024;                 // the vectors per channel stay in registers
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = kThreads == 32 ? lane : static_cast<int>(threadIdx.x);
  const long long workers = static_cast<long long>(gridDim.x) * kRows;
  const long long worker = static_cast<long long>(blockIdx.x) * kRows + (kRows > 1 ? warp : 0);
  long long row = worker * a.M / workers;
  const long long end = (worker + 1) * a.M / workers;
  if (row >= end) return;                                               // the same for all threads of a row
  const int C = a.C;
  uint32_t slot = 0;
  Slice hs[kJoin ? kVecs : 1], xs[kVecs];
  auto load = [&](long long at) {
    const bool live = at < end;
    if constexpr (kJoin) {
      const T* h = static_cast<const T*>(a.h) + at * a.h_stride;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) hs[i].load(h, i, t, C, live);
    }
    const T* x = static_cast<const T*>(a.x) + at * a.x_stride;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) xs[i].load(x, i, t, C, live);
  };
  load(row);
  float ja[8], jb[8], na[8], nb[8];
  long long group = -1, group_end = -1;
  for (; row < end; ++row) {
    if (row >= group_end) {
      group = a.rows_per_group > 0 ? row / a.rows_per_group : 0;
      group_end = a.rows_per_group > 0 ? (group + 1) * a.rows_per_group : a.M;
      if constexpr (kKeep) {
        if constexpr (kJoin) affine8<T, kMode, kThreads>(a.join, &a.gate, group, 0, t, C, ja, jb);
        if constexpr (kNext != kNextNone) affine8<T, kMode, kThreads>(a.norm, nullptr, group, 0, t, C, na, nb);
      }
    }
    float v[kVecs][8];
    float xv[kVecs][8];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      xs[i].get(kJoin ? xv[i] : v[i]);
      if constexpr (kJoin) hs[i].get(v[i]);
    }
    load(row + 1);
    if constexpr (kJoin) {
      norm_row<kMode, kThreads, kVecs>(a.join, v, C, t, smem, slot, lane, warp);
      T* r = static_cast<T*>(a.r) + row * a.r_stride;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        if constexpr (!kKeep) affine8<T, kMode, kThreads>(a.join, &a.gate, group, i, t, C, ja, jb);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] = OutTraits<T>::to_f(OutTraits<T>::from_f(fmaf(a.residual_scale, xv[i][j], fmaf(v[i][j], ja[j], jb[j]))));
          if (Slice::col(i, t, j) >= C) v[i][j] = 0.0f;
        }
        Slice::store(r, i, t, C, v[i]);
      }
    }
    if constexpr (kNext != kNextNone) {
      norm_row<kMode, kThreads, kVecs>(a.norm, v, C, t, smem, slot, lane, warp);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        if constexpr (!kKeep) affine8<T, kMode, kThreads>(a.norm, nullptr, group, i, t, C, na, nb);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf(v[i][j], na[j], nb[j]);
        if constexpr (kNext == kNextRows) {
          Slice::store(static_cast<T*>(a.y) + row * a.y_stride, i, t, C, v[i]);
        } else {
          const int col = Slice::col(i, t, 0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j >= C) v[i][j] = 0.0f;
          uint32_t word;
          const uint32_t codes = mx_quantize8(v[i], lane, word);     // the whole warp: blocks are shared by lanes
          if ((col >> 5) < a.blocks) *reinterpret_cast<uint32_t*>(a.codes + row * (16LL * a.blocks) + (col >> 1)) = codes;
          if ((lane & 15) == 0 && (col >> 7) < a.k_tiles)
            *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, col >> 7, a.k_tiles)) = word;
        }
      }
    }
  }
}

}  // namespace tb200
