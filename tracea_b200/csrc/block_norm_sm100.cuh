// The norm in front of a block and the join behind it, one pass over the rows:
//   join:  r = residual_scale * x + gate * (norm(h) * weight + bias) * (1 + scale) + shift ...   (the last two per group of rows)
//   norm:  y = (norm(r) * weight + bias) * (1 + scale) + shift, in the storage type or in the 4-bit format of mx_format.cuh
// with norm(v) = v / sqrt(mean(v^2) + eps) (rms), (v - mean) / sqrt(mean((v - mean)^2) + eps) (layer) or v (none). A call does either
// or both; the norm behind a join reads r as it is stored, so that both in one call give the bits of two calls.
//
// Bound by memory: a row is read once into registers, and everything is computed from there, in fp32. The second moment is taken
// about the mean in a pass of its own over the registers -- as mean(v^2) - mean^2 a row far from zero would lose it.
// A row belongs to a warp, or to all the threads of a CTA where it does not fit a warp's registers; a thread holds columns
// (i * threads + t) * 8 .. + 8, so that a warp's load covers 512 bytes, and four neighbouring lanes hold a block of the format.
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
  int vec;                  // all four matrices' rows are read and written eight elements at a time
  float residual_scale;
  NormVector gate;
  NormStage join, norm;
};

template <typename T>
__device__ __forceinline__ void norm_vector8(const NormVector& p, long long group, int col, int count, float (&v)[8]) {
  const long long at = group * p.group_stride + col;
  if (p.f32) {
    if (p.vec && count == 8) load8<float>(static_cast<const float*>(p.ptr) + at, v);
    else load8_upto<float>(static_cast<const float*>(p.ptr) + at, 1, count, v);
  } else {
    if (p.vec && count == 8) load8<T>(static_cast<const T*>(p.ptr) + at, v);
    else load8_upto<T>(static_cast<const T*>(p.ptr) + at, 1, count, v);
  }
}

template <int kThreads>
__device__ __forceinline__ float row_sum(float v, float* smem, int lane, int warp) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    __syncthreads();                       // the sums of the call before have been read
    if (lane == 0) smem[warp] = v;
    __syncthreads();
    v = lane < kWarps ? smem[lane] : 0.0f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  }
  return v;
}

// v, which holds the row with zeros past column C, becomes its norm, affine and modulated.
template <typename T, int kThreads, int kVecs>
__device__ __forceinline__ void norm_row(const NormStage& s, float (&v)[kVecs][8], int C, long long group, int t, float* smem,
                                         int lane, int warp) {
  float mean = 0.0f, inv = 1.0f;
  if (s.kind != kNormNone) {
    if (s.kind == kNormLayer) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[i][j];
      mean = row_sum<kThreads>(sum, smem, lane, warp) / static_cast<float>(C);
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int count = C - (i * kThreads + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mean;
        if (j < count) sq = fmaf(d, d, sq);
      }
    }
    inv = rsqrtf(row_sum<kThreads>(sq, smem, lane, warp) / static_cast<float>(C) + s.eps);
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = (i * kThreads + t) * 8;
    const int count = min(8, C - col);
    if (count <= 0) break;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - mean) * inv;
    float p[8];
    if (s.weight.ptr != nullptr) {
      norm_vector8<T>(s.weight, 0, col, count, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= p[j];
    }
    if (s.bias.ptr != nullptr) {
      norm_vector8<T>(s.bias, 0, col, count, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += p[j];
    }
    if (s.scale.ptr != nullptr) {
      norm_vector8<T>(s.scale, group, col, count, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = fmaf(v[i][j], p[j], v[i][j]);
    }
    if (s.shift.ptr != nullptr) {
      norm_vector8<T>(s.shift, group, col, count, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += p[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = j < count ? v[i][j] : 0.0f;
  }
}

__host__ __device__ constexpr int norm_block_threads(int row_threads) { return row_threads == 32 ? 256 : row_threads; }

template <typename T, int kThreads, int kVecs, bool kJoin, int kNext>
__global__ void __launch_bounds__(norm_block_threads(kThreads))
block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  __shared__ float smem[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kRows = norm_block_threads(kThreads) / kThreads;        // of a CTA
  const int t = kThreads == 32 ? lane : static_cast<int>(threadIdx.x);
  const long long stride = static_cast<long long>(gridDim.x) * kRows;
  for (long long row = static_cast<long long>(blockIdx.x) * kRows + (kRows > 1 ? warp : 0); row < a.M; row += stride) {
    const long long group = a.rows_per_group > 0 ? row / a.rows_per_group : 0;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float v[kVecs][8];
    if constexpr (kJoin) {
      const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
      float xv[kVecs][8];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = (i * kThreads + t) * 8;
        const int count = min(8, a.C - col);
        if (a.vec && count == 8) {
          load8<T>(h + col, v[i]);
          load8<T>(x + col, xv[i]);
        } else {
          load8_upto<T>(h + col, 1, count, v[i]);
          load8_upto<T>(x + col, 1, count, xv[i]);
        }
      }
      norm_row<T, kThreads, kVecs>(a.join, v, a.C, group, t, smem, lane, warp);
      T* r = static_cast<T*>(a.r) + row * a.r_stride;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = (i * kThreads + t) * 8;
        const int count = min(8, a.C - col);
        if (count <= 0) break;
        if (a.gate.ptr != nullptr) {
          float g[8];
          norm_vector8<T>(a.gate, group, col, count, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] *= g[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = OutTraits<T>::to_f(OutTraits<T>::from_f(fmaf(a.residual_scale, xv[i][j], v[i][j])));
        if (a.vec && count == 8) store8<T>(r + col, v[i]);
        else store8_upto<T>(r + col, 1, count, v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = (i * kThreads + t) * 8;
        const int count = min(8, a.C - col);
        if (a.vec && count == 8) load8<T>(x + col, v[i]);
        else load8_upto<T>(x + col, 1, count, v[i]);
      }
    }
    if constexpr (kNext != kNextNone) {
      norm_row<T, kThreads, kVecs>(a.norm, v, a.C, group, t, smem, lane, warp);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = (i * kThreads + t) * 8;
        const int count = min(8, a.C - col);
        if constexpr (kNext == kNextRows) {
          if (count <= 0) break;
          T* y = static_cast<T*>(a.y) + row * a.y_stride;
          if (a.vec && count == 8) store8<T>(y + col, v[i]);
          else store8_upto<T>(y + col, 1, count, v[i]);
        } else {
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
