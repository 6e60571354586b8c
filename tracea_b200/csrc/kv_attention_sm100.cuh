// What the kernels of attention over the cache share.
//
// One maximum serves the softmax and the values' scales: with s the score in powers of two and m >= s + ev for all tokens so far, up to
// a slack, the weights 2^(s + ev - m) need no scaling of v^ and fit halves, whatever the pages' scales are; the softmax's denominator
// is the sum of 2^(s + ev - m) 2^-ev. Since |ev| <= 40, neither can leave the range of fp32. The weights are halves because the matrix
// instructions take 16 bits of both operands; the denominator is summed from them before they are rounded. The slack: m moves only when a score
// passes it by 2^kSlack, so the sums are rescaled a few times a sequence and not every step.
#pragma once
#include "heads_sm100.cuh"

namespace tb200 {

constexpr float kSlack = 8.0f;
// Beyond 2^20 steps of fp32 are no longer small beside 1: there the maximum is taken from a score before anything is added to it, which is
// exact for scores near it, and follows it without slack, or weights would leave halves. A warp does so for all its rows if one has to.
constexpr float kFar = 1048576.0f;
constexpr float kLift = 7.0f;    // the weights are 2^7 times the above, up to 2^15: halves reach 2^16, and lose bits below 2^-14

struct KvAttentionArgs {
  CacheRef cache;
  SequencesRef seqs;
  const void* q;
  void* out;
  long long q_token, q_head, out_token, out_head;
  int q_vec;                     // q's heads can be read eight columns at a time
  int out_vec;                   // columns of out that can be written at a time: 8, 4 or 1
  int group;                     // heads of q to a head of keys
  int causal, window;
  int fewest, most;              // sequences with fewer or more rows (times group) are another kernel's
  int tile_rows, row_tiles;      // few rows: of a tile, and tiles of a sequence at most
  float scale_log2;              // |scale| * log2(e)
  float sign;                    // of the scale
  uint32_t* status;
  long long wait_limit;          // cycles any single wait may take before its role gives up
  int test_producer_stop;
};

__device__ __forceinline__ float exp2_ftz(float x) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
__device__ __forceinline__ float max_3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// An 8 x 8 matrix of halves, row lane / 4 and columns 2 (lane % 4) and the next in each lane, transposed.
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m != -INFINITY; }
// By what sums with the maximum m and the denominator l are taken in where the maximum of all is `top`: 0 for a part that has seen
// nothing, but for one that has seen nothing but NaN.
__device__ __forceinline__ float part_factor(float m, float l, float top) {
  return m == -INFINITY ? (l != l ? 1.0f : 0.0f) : exp2_ftz(m - top);
}
__device__ __forceinline__ void add_scaled(float4& sum, const float4& v, float f) {
  sum.x += f * v.x;
  sum.y += f * v.y;
  sum.z += f * v.z;
  sum.w += f * v.w;
}
// Four columns times `inv`; `vec` of them can be written at a time.
template <typename T>
__device__ __forceinline__ void store_4(T* p, const float4& v, float inv, int vec) {
  if (vec >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T, false>(v.x * inv, v.y * inv), pack2<T, false>(v.z * inv, v.w * inv));
  } else {
    p[0] = static_cast<T>(v.x * inv);
    p[1] = static_cast<T>(v.y * inv);
    p[2] = static_cast<T>(v.z * inv);
    p[3] = static_cast<T>(v.w * inv);
  }
}
// The power of two that brings a row whose largest absolute value is `peak` into [1, 2); 1 for a row of zeros or one that is not finite.
// `back` is its inverse. (Both within the normal range: peak 2^-127 and smaller, or 2^127 and larger, are not brought all the way.)
__device__ __forceinline__ float row_scale(float peak, float& back) {
  int e = static_cast<int>(__float_as_uint(peak) >> 23) - 127;
  if (peak == 0.0f || e == 128) e = 0;
  e = min(max(e, -126), 126);
  back = power_of_two(e);
  return power_of_two(-e);
}

}  // namespace tb200
