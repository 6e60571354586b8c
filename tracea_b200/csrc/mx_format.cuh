// The 4-bit microscaled format (OCP MX, E2M1 elements, E8M0 scales) as the kernels read and write it.
//
// A row's columns are cut into blocks of 32. A block holds 32 codes -- sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5,
// 2, 3, 4, 6 -- and one scale byte b that stands for 2^(b - 127), 255 for NaN. With p the block's largest absolute value,
//   b = clamp(floor(log2 p) - 2, -127, 125) + 127,   code = v / 2^(b - 127), to the nearest, ties to the even code, at most 6.
// Dividing by a power of two is exact, so the code is the only rounding. A block with a NaN or an infinity gets b = 255 and
// codes 0: it is NaN as a whole, since the elements cannot say which of them it was.
//
// Memory of an M x K matrix:
//   data    M rows of 16 * ceil(K / 32) bytes, the even column in a byte's low half; columns past K are 0
//   scales  ceil(M / 128) x ceil(K / 128) tiles of 512 bytes; row r, block b is byte 16 * (r % 32) + 4 * (r % 128 / 32) + b % 4 of
//           tile [r / 128][b / 4]: 32 lanes x 4 words, which tcgen05.cp takes to tensor memory as it is. Blocks past K are 0.
//           Rows past M are read, but reach no result.
#pragma once
#include <stdint.h>

#include "conv2d_sm100.cuh"

namespace tb200 {

constexpr int kMxBlock = 32;          // columns that share a scale
constexpr int kMxTileRows = 128;
constexpr int kMxTileCols = 128;      // 4 blocks
constexpr int kMxTileBytes = 512;

// Byte offset of the word with the scales of four blocks (columns 128 * kt ..) of row r.
__device__ __forceinline__ long long mx_scale_word(long long r, long long kt, long long k_tiles) {
  return ((r >> 7) * k_tiles + kt) * kMxTileBytes + 16 * (r & 31) + 4 * ((r & 127) >> 5);
}

// The scale byte of a block whose largest absolute value has the bits `peak`, and what its values are multiplied by.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t peak) {
  const uint32_t e = peak >> 23;                       // 0 for zero and subnormal values
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127)
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7fc00000u : byte << 23));
}

// Eight scaled values -> eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t mx_pack8(const float* v) {
  uint32_t r;
  asm("{\n"
      ".reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n"
      "}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight codes -> their values.
__device__ __forceinline__ void mx_unpack8(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n"
      ".reg .b8 a, b, c, d;\n"
      "mov.b32 {a, b, c, d}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n"
      "}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_abs8(const float* v) {
  return max_abs3(max_abs3(max_abs3(v[0], v[1], v[2]), v[3], v[4]), max_abs3(v[5], v[6], v[7]), 0.0f);
}
// The smallest of three, NaN if one of them is.
__device__ __forceinline__ float min_nan3(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Packed pairs: (a, b) * (c, d) [+ (e, f)].
__device__ __forceinline__ void mul2(float& a, float& b, float c, float d) {
  asm("{\n"
      ".reg .b64 x, y;\n"
      "mov.b64 x, {%0, %1};\n"
      "mov.b64 y, {%2, %3};\n"
      "mul.rn.f32x2 x, x, y;\n"
      "mov.b64 {%0, %1}, x;\n"
      "}\n"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ void fma2(float& a, float& b, float c, float d, float e, float f) {
  asm("{\n"
      ".reg .b64 x, y, z;\n"
      "mov.b64 x, {%0, %1};\n"
      "mov.b64 y, {%2, %3};\n"
      "mov.b64 z, {%4, %5};\n"
      "fma.rn.f32x2 x, x, y, z;\n"
      "mov.b64 {%0, %1}, x;\n"
      "}\n"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d), "f"(e), "f"(f));
}

// Quantises eight consecutive columns a lane, a block to four neighbouring lanes, all 32 lanes taking part: returns the lane's
// codes, and the block's scale byte in each of its four lanes.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&v)[8], uint32_t& byte) {
  float peak = max_abs8(v);
  peak = max_abs3(peak, __shfl_xor_sync(0xffffffffu, peak, 1), 0.0f);
  peak = max_abs3(peak, __shfl_xor_sync(0xffffffffu, peak, 2), 0.0f);
  byte = mx_scale_byte(__float_as_uint(peak));
  const float inv = mx_inverse(byte);
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    s[j] = v[j];
    s[j + 1] = v[j + 1];
    mul2(s[j], s[j + 1], inv, inv);
  }
  return byte == 255u ? 0u : mx_pack8(s);
}

// 32 consecutive columns in one thread -> 16 bytes of codes and the scale byte.
__device__ __forceinline__ uint4 mx_quantize32(const float (&v)[32], uint32_t& byte) {
  const float peak = max_abs3(max_abs3(max_abs8(v), max_abs8(v + 8), max_abs8(v + 16)), max_abs8(v + 24), 0.0f);
  byte = mx_scale_byte(__float_as_uint(peak));
  const float inv = mx_inverse(byte);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      s[j] = v[8 * q + j];
      s[j + 1] = v[8 * q + j + 1];
      mul2(s[j], s[j + 1], inv, inv);
    }
    w[q] = byte == 255u ? 0u : mx_pack8(s);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ReLU that keeps a NaN, so that a NaN block reaches the output whatever the epilogue (fmaxf would return the other operand).
__device__ __forceinline__ float relu_nan(float v) {
  float d;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(d) : "f"(v));
  return d;
}

// GELU of 16- and 4-bit outputs. (1 + tanh u) / 2 = 1 / (1 + e^-2u), which unlike the left side does not cancel for negative values:
// with tanh.approx (2^-11) results at -3 were off by a fifth. The exponent, in powers of two, is v (kGeluA + kGeluB v^2).
constexpr float kGeluA = -2.3022082f, kGeluB = -0.10294324f;      // -2 sqrt(2 / pi) log2(e), the same times 0.044715

// The activations of apply_act32 on one value, but for ReLU, which keeps NaN, and GELU.
template <bool kFast>
__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == kActRelu) return relu_nan(v);
  if (act == kActSilu) {
    if constexpr (kFast) return __fdividef(v, 1.0f + __expf(-v));
    else return v / (1.0f + expf(-v));
  }
  if (act == kActGelu) {
    if constexpr (kFast) {
      float t = v * fmaf(kGeluB, v * v, kGeluA);
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t));
      return __fdividef(v, 1.0f + t);
    } else {
      const float u = 0.79788456f * (v + 0.044715f * v * v * v);
      return 0.5f * v * (1.0f + tanhf(u));
    }
  }
  return v;
}

// Eight consecutive elements as fp32: `p` at the first one, 16 (32 for fp32) aligned bytes, or element by element.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    unpack2<T>(a.x, v[0], v[1]);
    unpack2<T>(a.y, v[2], v[3]);
    unpack2<T>(a.z, v[4], v[5]);
    unpack2<T>(a.w, v[6], v[7]);
  }
}
template <typename T>
__device__ __forceinline__ void load8_upto(const T* p, long long step, int count, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < count ? OutTraits<T>::to_f(p[j * step]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T, false>(v[0], v[1]), pack2<T, false>(v[2], v[3]),
                                              pack2<T, false>(v[4], v[5]), pack2<T, false>(v[6], v[7]));
  }
}
template <typename T>
__device__ __forceinline__ void store8_upto(T* p, long long step, int count, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) p[j * step] = OutTraits<T>::from_f(v[j]);
}

// ------------------------------------------------------------------ matrix <-> format
struct MxCopyArgs {
  const void* src;       // quantise: the matrix; dequantise: the codes
  void* dst;
  void* scales;
  long long row_stride, col_stride;   // of the matrix, in elements
  long long M;
  int K, blocks, k_tiles;
  int chunks;            // of 256 columns
};

constexpr int kMxCopyThreads = 256;

// A warp takes 256 columns of four rows 32 apart, whose scales are 16 consecutive bytes a tile. One pass: bytes in and bytes out.
// kVec: rows are read in 16-byte accesses, K a multiple of 8; the four rows' loads are in flight together.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kMxCopyThreads)
mx_quantize_kernel(const __grid_constant__ MxCopyArgs a) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * (kMxCopyThreads / 32) + (threadIdx.x >> 5);
  const long long rows32 = task / a.chunks;
  const int chunk = static_cast<int>(task - rows32 * a.chunks);
  const long long r0 = (rows32 >> 5) * 128 + (rows32 & 31);
  if (r0 - (r0 & 127) >= a.M) return;                    // warp-uniform
  const int col = chunk * 256 + lane * 8;
  const int count = min(8, a.K - col);
  const T* src = static_cast<const T*>(a.src) + r0 * a.row_stride + col * a.col_stride;
  uint4 raw[kVec ? 4 : 1][sizeof(T) / 2];
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q)
        raw[i][q] = r0 + 32 * i < a.M && count > 0 ? reinterpret_cast<const uint4*>(src + 32 * i * a.row_stride)[q]
                                                   : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t words[4];
  uint8_t* dst = static_cast<uint8_t*>(a.dst) + r0 * (16LL * a.blocks) + (col >> 1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
    if constexpr (kVec) load8<T>(reinterpret_cast<const T*>(raw[i]), v);
    else load8_upto<T>(src + 32 * i * a.row_stride, a.col_stride, r0 + 32 * i < a.M ? count : 0, v);
    const uint32_t codes = mx_quantize8(v, words[i]);
    words[i] <<= 8 * ((lane >> 2) & 3);                  // the word of four blocks, of 16 lanes
    words[i] |= __shfl_xor_sync(0xffffffffu, words[i], 4);
    words[i] |= __shfl_xor_sync(0xffffffffu, words[i], 8);
    if (r0 + 32 * i < a.M && (col >> 5) < a.blocks) *reinterpret_cast<uint32_t*>(dst + 32 * i * (16LL * a.blocks)) = codes;
  }
  if ((lane & 15) == 0 && (col >> 7) < a.k_tiles)
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.scales) + mx_scale_word(r0, col >> 7, a.k_tiles)) =
        make_uint4(words[0], words[1], words[2], words[3]);
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kMxCopyThreads)
mx_dequantize_kernel(const __grid_constant__ MxCopyArgs a) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * (kMxCopyThreads / 32) + (threadIdx.x >> 5);
  const long long rows32 = task / a.chunks;
  const int chunk = static_cast<int>(task - rows32 * a.chunks);
  const long long r0 = (rows32 >> 5) * 128 + (rows32 & 31);
  const int col = chunk * 256 + lane * 8;
  const int count = min(8, a.K - col);
  if (r0 >= a.M || count <= 0) return;
  const uint4 words = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.scales) + mx_scale_word(r0, col >> 7, a.k_tiles));
  const uint32_t word[4] = {words.x, words.y, words.z, words.w};
  const uint8_t* src = static_cast<const uint8_t*>(a.src) + r0 * (16LL * a.blocks) + (col >> 1);
  T* dst = static_cast<T*>(a.dst) + r0 * a.row_stride + col * a.col_stride;
  uint32_t codes[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    codes[i] = r0 + 32 * i < a.M ? *reinterpret_cast<const uint32_t*>(src + 32 * i * (16LL * a.blocks)) : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r0 + 32 * i >= a.M) break;
    const float s = mx_scale_value((word[i] >> (8 * ((col >> 5) & 3))) & 255u);
    float v[8];
    mx_unpack8(codes[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s;
    if constexpr (kVec) store8<T>(dst + 32 * i * a.row_stride, v);
    else store8_upto<T>(dst + 32 * i * a.row_stride, a.col_stride, count, v);
  }
}

}  // namespace tb200
