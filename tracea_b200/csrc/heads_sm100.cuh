// Rows of heads on their way into attention: the norm of a head's columns, the rotation of its pairs of columns by the token's
// position, and the cache of keys and values in 8 bits.
//
// All of it is bound by reading and writing the rows once. A row of D columns is held by a few lanes, 16 columns each, so that the
// norm is a few shuffles and the pairs of a rotation lie in one lane; the angles, which all heads of a token share, are computed
// once for them: they are the only arithmetic that would weigh.
//
// The cache (TraceaKvCache): a block is the P x D elements of a page and head, of keys or of values, row by row, in e4m3, and a
// byte b that scales them by 2^(b - 127). Powers of two: an element is rounded once, by its own mantissa, and when a block's scale
// grows behind it, its older elements move by a power of two, which changes only those that leave the normal range.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx_format.cuh"
#include "ptx_sm100.cuh"

namespace tb200 {

constexpr int kHeadThreads = 256;
constexpr int kHeadMaxColumns = 256;
constexpr int kCacheMaxColumns = 128;
constexpr int kCacheMaxPage = 128;
constexpr int kMaxTokens = 1 << 30;        // of a sequence
constexpr long long kCacheMostQueryHeads = 1 << 23;   // times the rows of a page: 2^30, which kv_append_kernel counts in 32 bits
constexpr int kCacheMinExponent = -40, kCacheMaxExponent = 40;

struct Rotation {
  const double* frequencies;   // angle per position of a pair, in radians
  int pairs;                   // 0: no rotation
  int interleaved;             // pair i is columns 2i and 2i + 1; else i and i + pairs
};

// Cosine and sine of position * frequency. The angle is taken in turns and in 64 bits, and so are the quarter turns that are cut off:
// fp32 would be off by 2^-24 of an angle that grows with the position. Of what is left, x within +-pi/4, the Taylor polynomials up to
// x^9 and x^10, whose next terms are below 2^-29 and 2^-31.
struct Angle {
  double quarters;                      // a step's, in quarter turns
  __device__ __forceinline__ explicit Angle(double frequency) : quarters(frequency * 0.63661977236758134308) {}   // 2 / pi
  __device__ __forceinline__ void turn(double position, float& c, float& s) const {
    constexpr double kWhole = 6755399441055744.0;        // 1.5 * 2^52: adding it leaves a whole number in the low bits
    const double all = position * quarters, whole = all + kWhole;
    const int quadrant = __double2loint(whole);
    const float x = static_cast<float>(all - (whole - kWhole)) * 1.57079633f, z = x * x;
    float sine = fmaf(z, 1.0f / 362880, -1.0f / 5040), cosine = fmaf(z, -1.0f / 3628800, 1.0f / 40320);
    sine = fmaf(z, sine, 1.0f / 120);
    cosine = fmaf(z, cosine, -1.0f / 720);
    sine = fmaf(z, sine, -1.0f / 6);
    cosine = fmaf(z, cosine, 1.0f / 24);
    sine = fmaf(x * z, sine, x);
    cosine = fmaf(z, cosine, -0.5f);
    cosine = fmaf(z, cosine, 1.0f);
    c = (quadrant & 1) ? sine : cosine;
    s = (quadrant & 1) ? cosine : sine;
    if ((quadrant + 1) & 2) c = -c;
    if (quadrant & 2) s = -s;
  }
};

// ------------------------------------------------------------------ a lane's columns of a row
// A lane holds kPairs pairs (x, y) of columns, which a rotation turns into (x cos - y sin, y cos + x sin).
// kLanes > 0: so many lanes hold a row, 8 pairs each, 16 columns in two runs of 8: 8c and 8c + pairs for lane c, which a rotation of
// halves pairs, for the rotated columns of that kind; 16c and 16c + 8 for others. Rows are 16-byte aligned, D and the rotated columns
// multiples of 16.
// kLanes = 0: a warp holds a row of any even number of columns, a lane the pairs number lane + 32 i.
__host__ __device__ constexpr int head_row_lanes(int lanes) { return lanes > 0 ? lanes : 32; }
template <int kLanes, int kScalarPairs>
struct HeadLane {
  static constexpr bool kVec = kLanes > 0;
  static constexpr int kPairs = kVec ? 8 : kScalarPairs;
  int first[kVec ? 1 : kPairs], second[kVec ? 1 : kPairs];   // columns; 0, 0 where there are none
  int angle;                                                 // number of the first pair's angle
  int live;                                                  // pairs that there are
  bool turned;

  __device__ __forceinline__ HeadLane(int lane, int D, const Rotation& rot) {
    if constexpr (kVec) {
      live = 16 * lane < D ? kPairs : 0;
      turned = 16 * lane < 2 * rot.pairs;
      angle = 8 * lane;
      const bool halves = turned && rot.interleaved == 0;
      first[0] = live == 0 ? 0 : halves ? 8 * lane : 16 * lane;
      second[0] = live == 0 ? 0 : halves ? 8 * lane + rot.pairs : 16 * lane + 8;
    } else {
      turned = true;
      angle = lane;
      live = 0;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int p = lane + 32 * i;
        const bool halves = p < rot.pairs && rot.interleaved == 0;
        if (2 * p < D) live = i + 1;
        first[i] = 2 * p >= D ? 0 : halves ? p : 2 * p;
        second[i] = 2 * p >= D ? 0 : halves ? p + rot.pairs : 2 * p + 1;
      }
    }
  }
};

// Between the order of the runs in memory and that of pairs of neighbours.
__device__ __forceinline__ void runs_to_pairs(float (&x)[8], float (&y)[8]) {
  const float a[8] = {x[0], x[2], x[4], x[6], y[0], y[2], y[4], y[6]}, b[8] = {x[1], x[3], x[5], x[7], y[1], y[3], y[5], y[7]};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = a[i];
    y[i] = b[i];
  }
}
__device__ __forceinline__ void pairs_to_runs(float (&x)[8], float (&y)[8]) {
  const float a[8] = {x[0], y[0], x[1], y[1], x[2], y[2], x[3], y[3]}, b[8] = {x[4], y[4], x[5], y[5], x[6], y[6], x[7], y[7]};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = a[i];
    y[i] = b[i];
  }
}

template <typename T>
struct Vec8 {   // eight consecutive elements as they are loaded
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void fetch8(const T* p, Vec8<T>& v) {
  v.w[0] = *reinterpret_cast<const uint4*>(p);
  if constexpr (sizeof(T) == 4) v.w[1] = *reinterpret_cast<const uint4*>(p + 4);
}
template <typename T>
__device__ __forceinline__ void widen8(const Vec8<T>& v, float (&o)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float* e = reinterpret_cast<const float*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = e[i];
  } else {
    unpack2<T>(v.w[0].x, o[0], o[1]);
    unpack2<T>(v.w[0].y, o[2], o[3]);
    unpack2<T>(v.w[0].z, o[4], o[5]);
    unpack2<T>(v.w[0].w, o[6], o[7]);
  }
}

// A lane's columns of a row as they lie in memory. Lanes without columns, and those whose row is not one, load some other of the same
// tensor: a branch around a load costs more.
template <typename T, int kLanes, int kScalarPairs>
struct HeadRaw {
  using Lane = HeadLane<kLanes, kScalarPairs>;
  static constexpr int kPairs = Lane::kPairs;
  Vec8<T> va, vb;
  T sa[kScalarPairs], sb[kScalarPairs];

  __device__ __forceinline__ void load(const T* row, const Lane& l) {
    if constexpr (Lane::kVec) {
      fetch8(row + l.first[0], va);
      fetch8(row + l.second[0], vb);
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        sa[i] = row[l.first[i]];
        sb[i] = row[l.second[i]];
      }
    }
  }
  template <bool kNeighbours>
  __device__ __forceinline__ void values(const Lane& l, float (&x)[kPairs], float (&y)[kPairs]) const {
    if constexpr (Lane::kVec) {
      widen8(va, x);
      widen8(vb, y);
      if constexpr (kNeighbours) runs_to_pairs(x, y);
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        x[i] = i < l.live ? static_cast<float>(sa[i]) : 0.0f;
        y[i] = i < l.live ? static_cast<float>(sb[i]) : 0.0f;
      }
    }
  }
};

template <bool kNeighbours, typename T, int kLanes, int kScalarPairs>
__device__ __forceinline__ void head_store(T* row, const HeadLane<kLanes, kScalarPairs>& l, float (&x)[HeadLane<kLanes, kScalarPairs>::kPairs],
                                           float (&y)[HeadLane<kLanes, kScalarPairs>::kPairs]) {
  if constexpr (kLanes > 0) {
    if constexpr (kNeighbours) pairs_to_runs(x, y);
    if (l.live > 0) {
      store8(row + l.first[0], x);
      store8(row + l.second[0], y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScalarPairs; ++i) {
      if (i < l.live) {
        row[l.first[i]] = static_cast<T>(x[i]);
        row[l.second[i]] = static_cast<T>(y[i]);
      }
    }
  }
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 1 / sqrt(mean + eps) of a row, to 2 units in the last place.
template <int kLanes, int kScalarPairs>
__device__ __forceinline__ float head_norm(const HeadLane<kLanes, kScalarPairs>& l, const float (&x)[HeadLane<kLanes, kScalarPairs>::kPairs],
                                           const float (&y)[HeadLane<kLanes, kScalarPairs>::kPairs], float inv_columns, float eps) {
  constexpr int kPairs = HeadLane<kLanes, kScalarPairs>::kPairs;
  uint64_t both = 0;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const uint64_t v = pack_f32x2(x[i], y[i]);
    both = fma_f32x2(v, v, both);
  }
  float sum, other;
  unpack_f32x2(both, sum, other);
  sum = l.live > 0 ? sum + other : 0.0f;
#pragma unroll
  for (int o = head_row_lanes(kLanes) / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return rsqrtf(sum * inv_columns + eps);
}

// A lane's weights, 1 where there are none; `weight`: fp32 in shared memory, or nullptr.
template <bool kNeighbours, int kLanes, int kScalarPairs>
__device__ __forceinline__ void head_weights(const HeadLane<kLanes, kScalarPairs>& l, const float* weight,
                                             float (&wx)[HeadLane<kLanes, kScalarPairs>::kPairs], float (&wy)[HeadLane<kLanes, kScalarPairs>::kPairs]) {
  if (weight == nullptr) {
#pragma unroll
    for (int i = 0; i < HeadLane<kLanes, kScalarPairs>::kPairs; ++i) wx[i] = wy[i] = 1.0f;
  } else if constexpr (kLanes > 0) {
    load8(weight + l.first[0], wx);
    load8(weight + l.second[0], wy);
    if constexpr (kNeighbours) runs_to_pairs(wx, wy);
  } else {
#pragma unroll
    for (int i = 0; i < kScalarPairs; ++i) {
      wx[i] = weight[l.first[i]];
      wy[i] = weight[l.second[i]];
    }
  }
}
// A lane's cosines and sines; `turns`: a token's, those of all pairs and then these, in shared memory.
template <int kLanes, int kScalarPairs>
__device__ __forceinline__ void head_turns(const HeadLane<kLanes, kScalarPairs>& l, const float* turns, int pairs,
                                           float (&c)[HeadLane<kLanes, kScalarPairs>::kPairs], float (&s)[HeadLane<kLanes, kScalarPairs>::kPairs]) {
#pragma unroll
  for (int i = 0; i < HeadLane<kLanes, kScalarPairs>::kPairs; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if constexpr (kLanes > 0) {
    if (l.turned) {
      load8(turns + l.angle, c);
      load8(turns + pairs + l.angle, s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScalarPairs; ++i) {
      if (l.angle + 32 * i < pairs) {
        c[i] = turns[l.angle + 32 * i];
        s[i] = turns[pairs + l.angle + 32 * i];
      }
    }
  }
}
// Weights and rotation together, for rows of one token: (x, y) -> factor (x xx + y xy, y yy + x yx), two pairs at a time. Columns that are
// not rotated are only multiplied: 0 times a partner that is not finite would be NaN.
template <int kPairs>
struct HeadTurn {
  uint64_t xx[kPairs / 2], xy[kPairs / 2], yy[kPairs / 2], yx[kPairs / 2];
  __device__ __forceinline__ HeadTurn(const float (&wx)[kPairs], const float (&wy)[kPairs], const float (&c)[kPairs], const float (&s)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      const int a = 2 * i, b = 2 * i + 1;
      xx[i] = pack_f32x2(wx[a] * c[a], wx[b] * c[b]);
      xy[i] = pack_f32x2(-wy[a] * s[a], -wy[b] * s[b]);
      yy[i] = pack_f32x2(wy[a] * c[a], wy[b] * c[b]);
      yx[i] = pack_f32x2(wx[a] * s[a], wx[b] * s[b]);
    }
  }
  // pairs: those of the whole rotation
  template <typename Lane>
  __device__ __forceinline__ void apply(const Lane& l, int pairs, float (&x)[kPairs], float (&y)[kPairs], float factor) const {
    const uint64_t f = pack_f32x2(factor, factor);
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      const uint64_t u = mul_f32x2(pack_f32x2(x[2 * i], x[2 * i + 1]), f), v = mul_f32x2(pack_f32x2(y[2 * i], y[2 * i + 1]), f);
      uint64_t a = mul_f32x2(u, xx[i]), b = mul_f32x2(v, yy[i]);
      if constexpr (Lane::kVec) {
        if (l.turned) {
          a = fma_f32x2(v, xy[i], a);
          b = fma_f32x2(u, yx[i], b);
        }
        unpack_f32x2(a, x[2 * i], x[2 * i + 1]);
        unpack_f32x2(b, y[2 * i], y[2 * i + 1]);
      } else {
        float p[4], q[4];                                    // multiplied only, rotated
        unpack_f32x2(a, p[0], p[1]);
        unpack_f32x2(b, p[2], p[3]);
        unpack_f32x2(fma_f32x2(v, xy[i], a), q[0], q[1]);
        unpack_f32x2(fma_f32x2(u, yx[i], b), q[2], q[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool turned = l.angle + 32 * (2 * i + j) < pairs;
          x[2 * i + j] = turned ? q[j] : p[j];
          y[2 * i + j] = turned ? q[2 + j] : p[2 + j];
        }
      }
    }
  }
};

// ------------------------------------------------------------------ norm and rotation of rows of heads
struct HeadRows {
  const void* x;
  void* y;
  const void* weight;
  int weight_f32;
  int heads;
  long long x_token, x_head, y_token, y_head;   // strides in elements
};

struct HeadRotateArgs {
  HeadRows rows[2];            // queries, keys
  Rotation rot;
  const int* positions;
  int tokens, D, norm;
  int passes;                  // of a warp, over as many heads as it holds, that a token takes in all; blockIdx.y shares them out
  float eps;
};

template <typename T>
__device__ __forceinline__ void weights_to_shared(float* dst, const void* weight, int is_f32, int D) {
  if (weight == nullptr) return;
  for (int i = threadIdx.x; i < D; i += kHeadThreads)
    dst[i] = is_f32 ? static_cast<const float*>(weight)[i] : static_cast<float>(static_cast<const T*>(weight)[i]);
}

// A warp takes as many of a token's heads as it holds at a time, queries and then keys, or, where the tokens alone would not fill the
// machine, a share of them. The weights and the token's rotation stay in registers over them; kAhead passes' loads are under way at once.
template <typename T, int kLanes, bool kNeighbours>
__global__ void __launch_bounds__(kHeadThreads, 3) head_rotate_kernel(const __grid_constant__ HeadRotateArgs args) {
  using Lane = HeadLane<kLanes, 4>;
  constexpr int kPairs = Lane::kPairs, kRowLanes = head_row_lanes(kLanes), kHeads = 32 / kRowLanes, kAhead = 2;
  __shared__ __align__(16) float weights[2][kHeadMaxColumns];
  __shared__ __align__(16) float turns[kHeadThreads / 32][kHeadMaxColumns];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long token = static_cast<long long>(blockIdx.x) * (kHeadThreads / 32) + warp;
  for (int r = 0; r < 2; ++r) weights_to_shared<T>(weights[r], args.rows[r].weight, args.rows[r].weight_f32, args.D);
  if (token < args.tokens && args.rot.pairs > 0) {
    const double position = args.positions[token];
    for (int p = lane; p < args.rot.pairs; p += 32) Angle(args.rot.frequencies[p]).turn(position, turns[warp][p], turns[warp][args.rot.pairs + p]);
  }
  __syncthreads();
  if (token >= args.tokens) return;
  const int group = lane / kRowLanes;
  const Lane l(lane % kRowLanes, args.D, args.rot);
  const float inv_columns = 1.0f / static_cast<float>(args.D);
  float c[kPairs], s[kPairs];
  head_turns(l, turns[warp], args.rot.pairs, c, s);
  const int split_begin = args.passes * static_cast<int>(blockIdx.y) / static_cast<int>(gridDim.y);
  const int split_end = args.passes * static_cast<int>(blockIdx.y + 1) / static_cast<int>(gridDim.y);
  int before = 0;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const HeadRows& rows = args.rows[which];
    const int passes = (rows.heads + kHeads - 1) / kHeads;
    const int begin = max(0, split_begin - before), end = min(passes, split_end - before);
    before += passes;
    if (begin >= end) continue;
    float wx[kPairs], wy[kPairs];
    head_weights<kNeighbours>(l, rows.weight != nullptr ? weights[which] : nullptr, wx, wy);
    const HeadTurn<kPairs> turn(wx, wy, c, s);
    const int heads = rows.heads;
    const long long x_step = kHeads * rows.x_head, y_step = kHeads * rows.y_head;
    const T* src = static_cast<const T*>(rows.x) + token * rows.x_token + (begin * kHeads + group) * rows.x_head;
    T* dst = static_cast<T*>(rows.y) + token * rows.y_token + (begin * kHeads + group) * rows.y_head;
    const T* const some = static_cast<const T*>(rows.x) + token * rows.x_token;
    for (int pass = begin; pass < end; pass += kAhead) {
      HeadRaw<T, kLanes, 4> raw[kAhead];
      bool here[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        here[u] = pass + u < end && (pass + u) * kHeads + group < heads;
        raw[u].load(here[u] ? src + u * x_step : some, l);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float x[kPairs], y[kPairs];
        raw[u].template values<kNeighbours>(l, x, y);
        turn.apply(l, args.rot.pairs, x, y, args.norm ? head_norm(l, x, y, inv_columns, args.eps) : 1.0f);
        if (here[u]) head_store<kNeighbours>(dst + u * y_step, l, x, y);
      }
      src += kAhead * x_step;
      dst += kAhead * y_step;
    }
  }
}

// ------------------------------------------------------------------ the cache
struct CacheRef {
  uint8_t *k, *v, *k_scales, *v_scales;
  long long pages;
  int heads, page_shift, D;
};
// Sequence s has `lengths[s]` tokens, the last starts[s + 1] - starts[s] of which are the rows from starts[s] on (starts nullptr: the
// last one is row s). Token j lies in row j % P of page table[s][j / P]; an entry that is no page, and what the table is too short
// for, holds no tokens.
struct SequencesRef {
  const int *table, *lengths, *starts;
  long long table_stride;
  int table_width, count, rows;
};

// Item number `index` of all sequences' items in line, `items(rows, length)` of each that has rows; found by a whole warp, 32 sequences
// at a time. False past the last one. Whatever lengths and starts hold, the rows found are rows.
struct SequenceItem {
  int sequence, item, first_row, rows, length;
};
template <typename Items>
__device__ __forceinline__ bool find_sequence(const SequencesRef& s, int index, SequenceItem& found, Items&& items) {
  const int lane = threadIdx.x & 31;
  if (s.starts == nullptr) {           // a row each, and so an item
    if (index >= s.count) return false;
    found = {index, 0, index, 1, max(0, min(s.lengths[index], kMaxTokens))};
    return true;
  }
  int before = 0;
  for (int base = 0; base < s.count; base += 32) {
    const int i = base + lane;
    int row = 0, n = 0, length = 0, mine = 0;
    if (i < s.count) {
      row = max(0, min(s.starts[i], s.rows));
      n = max(0, min(s.starts[i + 1], s.rows) - row);
      length = max(0, min(s.lengths[i], kMaxTokens));
      mine = n > 0 ? items(n, length) : 0;
    }
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + sum > index);
    if (past != 0u) {
      const int at = __ffs(static_cast<int>(past)) - 1;
      found.sequence = base + at;
      found.item = index - before - __shfl_sync(0xffffffffu, sum - mine, at);
      found.first_row = __shfl_sync(0xffffffffu, row, at);
      found.rows = __shfl_sync(0xffffffffu, n, at);
      found.length = __shfl_sync(0xffffffffu, length, at);
      return true;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

// The smallest e of which 448 2^e reach `peak` >= 0, within the format's range: 448 is 1.75 * 2^8.
__device__ __forceinline__ int cache_exponent(float peak) {
  const uint32_t u = __float_as_uint(peak);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kCacheMinExponent), kCacheMaxExponent);
}

// Two elements, to nearest even, saturated; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) { return e4m3_pair(a, b) | (e4m3_pair(c, d) << 16); }
__device__ __forceinline__ uint2 e4m3_eight(const float (&v)[8]) {
  return make_uint2(e4m3_four(v[0], v[1], v[2], v[3]), e4m3_four(v[4], v[5], v[6], v[7]));
}
// Four elements as halves, two to a word.
__device__ __forceinline__ void halves_of_e4m3(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n"
      ".reg .b16 l, h;\n"
      "mov.b32 {l, h}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ uint32_t e4m3_rescaled(uint32_t four, float factor) {
  uint32_t lo, hi;
  halves_of_e4m3(four, lo, hi);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return e4m3_four(x.x * factor, x.y * factor, y.x * factor, y.y * factor);
}

// ------------------------------------------------------------------ appending to the cache
struct KvAppendArgs {
  CacheRef cache;
  SequencesRef seqs;
  HeadRows q, k;               // q.x may be nullptr; k has no y
  const void* v;
  long long v_token, v_head;
  Rotation rot;
  int norm;
  int group;                   // heads of q to one of k
  int heads_per_cta;           // of k
  int turn_rows;               // rows of angles in shared memory
  int turn_lanes;              // threads that compute a row of them: a power of two, at least its pairs
  float eps;
};

// A CTA takes the new tokens of one page of a sequence, and some heads: for each the keys and values, whose scales need all of the
// block's rows and so stay in registers until they are known, and the queries' heads that go with it. A block belongs to one CTA:
// nothing is shared, nothing atomic. kRows: rows of a block that a lane holds.
template <typename T, int kLanes, bool kNeighbours, int kRows>
__global__ void __launch_bounds__(kHeadThreads, kLanes > 0 && kRows <= 2 ? 2 : 1) kv_append_kernel(const __grid_constant__ KvAppendArgs args) {
  constexpr int kScalarPairs = kCacheMaxColumns / 64;
  using Lane = HeadLane<kLanes, kScalarPairs>;
  using Raw = HeadRaw<T, kLanes, kScalarPairs>;
  constexpr int kPairs = Lane::kPairs, kWarps = kHeadThreads / 32, kRowLanes = head_row_lanes(kLanes), kRowsAtOnce = kHeadThreads / kRowLanes;
  extern __shared__ __align__(16) float turns[];           // [turn_rows][2][pairs]: cosines, sines
  __shared__ __align__(16) float weights[2][kCacheMaxColumns];
  __shared__ float peaks[2][2][kWarps];                    // two heads in turn: one barrier a head
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int shift = args.cache.page_shift, D = args.cache.D;
  SequenceItem at;
  const bool any = find_sequence(args.seqs, static_cast<int>(blockIdx.x), at, [&](int n, int length) {
    return ((length - 1) >> shift) - ((length - n) >> shift) + 1;
  });
  if (!any) return;
  const int begin = at.length - at.rows;                   // position of the sequence's first new token
  const int slot = (begin >> shift) + at.item;
  const int from = max(begin, slot << shift), to = min(at.length, (slot + 1) << shift);
  const int count = to - from, first = from - (slot << shift);
  const int row0 = at.first_row + from - begin;
  int entry = -1;                                          // looked at below, when it has arrived
  if (slot >= 0 && slot < args.seqs.table_width) entry = args.seqs.table[at.sequence * args.seqs.table_stride + slot];

  const int my_row = static_cast<int>(threadIdx.x) / kRowLanes, my_lane = static_cast<int>(threadIdx.x) % kRowLanes;
  const Lane l(my_lane, D, args.rot);
  const Lane plain(my_lane, D, Rotation{nullptr, 0, 0});   // values are not rotated: their columns in order
  const float inv_columns = 1.0f / static_cast<float>(D);
  const int head0 = static_cast<int>(blockIdx.y) * args.heads_per_cta, head1 = min(args.cache.heads, head0 + args.heads_per_cta);

  // the first head's keys and values, on their way while the angles are computed
  Raw rk[kRows], rv[kRows];
  const T *k_row[kRows], *v_row[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = my_row + i * kRowsAtOnce;
    const long long row = row0 + (r < count ? r : 0);
    k_row[i] = static_cast<const T*>(args.k.x) + row * args.k.x_token + head0 * args.k.x_head;
    v_row[i] = static_cast<const T*>(args.v) + row * args.v_token + head0 * args.v_head;
    rk[i].load(k_row[i], l);
    rv[i].load(v_row[i], plain);
  }

  weights_to_shared<T>(weights[0], args.q.weight, args.q.weight_f32, D);
  weights_to_shared<T>(weights[1], args.k.weight, args.k.weight_f32, D);
  const int pairs = args.rot.pairs;
  const int my_pair = static_cast<int>(threadIdx.x) & (args.turn_lanes - 1);
  if (my_pair < pairs) {
    const Angle angle(args.rot.frequencies[my_pair]);
    const int step = kHeadThreads / args.turn_lanes;
    for (int r = static_cast<int>(threadIdx.x) / args.turn_lanes; r < count; r += step)
      angle.turn(from + r, turns[2 * r * pairs + my_pair], turns[(2 * r + 1) * pairs + my_pair]);
  }
  __syncthreads();

  const long long page = entry >= 0 && entry < args.cache.pages ? entry : -1;
  if (page >= 0) {
    for (int head = head0; head < head1; ++head) {
      const long long block = page * args.cache.heads + head;
      uint8_t* ck = args.cache.k + (block << shift) * D;
      uint8_t* cv = args.cache.v + (block << shift) * D;
      const int old_k = static_cast<int>(args.cache.k_scales[block]) - 127, old_v = static_cast<int>(args.cache.v_scales[block]) - 127;
      float kx[kRows][kPairs], ky[kRows][kPairs];
      float peak_k = 0.0f, peak_v = 0.0f;
      uint32_t bad = 0u;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = my_row + i * kRowsAtOnce;
        rk[i].template values<kNeighbours>(l, kx[i], ky[i]);
        float wx[kPairs], wy[kPairs];
        head_weights<kNeighbours>(l, args.k.weight != nullptr ? weights[1] : nullptr, wx, wy);
        const float factor = args.norm ? head_norm(l, kx[i], ky[i], inv_columns, args.eps) : 1.0f;
        float c[kPairs], s[kPairs];
        head_turns(l, turns + 2 * (r < count ? r : 0) * pairs, pairs, c, s);
        float mk = 0.0f, mv = 0.0f;                        // NaN if there is one among them
#pragma unroll
        for (int j = 0; j < kPairs; j += 2) {
          const uint64_t f = pack_f32x2(factor, factor), co = pack_f32x2(c[j], c[j + 1]), si = pack_f32x2(s[j], s[j + 1]);
          const uint64_t x = mul_f32x2(mul_f32x2(pack_f32x2(kx[i][j], kx[i][j + 1]), f), pack_f32x2(wx[j], wx[j + 1]));
          const uint64_t y = mul_f32x2(mul_f32x2(pack_f32x2(ky[i][j], ky[i][j + 1]), f), pack_f32x2(wy[j], wy[j + 1]));
          unpack_f32x2(fma_f32x2(y, pack_f32x2(-s[j], -s[j + 1]), mul_f32x2(x, co)), kx[i][j], kx[i][j + 1]);
          unpack_f32x2(fma_f32x2(x, si, mul_f32x2(y, co)), ky[i][j], ky[i][j + 1]);
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j) mk = max_nan(mk, max_nan(fabsf(kx[i][j]), fabsf(ky[i][j])));
        float vx[kPairs], vy[kPairs];
        rv[i].template values<false>(plain, vx, vy);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) mv = max_nan(mv, max_nan(fabsf(vx[j]), fabsf(vy[j])));
        if (l.live == 0 || r >= count) mk = mv = 0.0f;
        // a token that is not finite counts for no scale: a vote of its lanes
        const uint32_t votes = __ballot_sync(0xffffffffu, !(mk < INFINITY && mv < INFINITY));
        const uint32_t mine = kRowLanes == 32 ? votes : (votes >> ((threadIdx.x & 31) / kRowLanes * kRowLanes)) & ((1u << (kRowLanes % 32)) - 1u);
        if (mine != 0u) bad |= 1u << i;
        else {
          peak_k = fmaxf(peak_k, mk);
          peak_v = fmaxf(peak_v, mv);
        }
      }
      if (head + 1 < head1) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) rk[i].load(k_row[i] += args.k.x_head, l);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        peak_k = fmaxf(peak_k, __shfl_xor_sync(0xffffffffu, peak_k, o));
        peak_v = fmaxf(peak_v, __shfl_xor_sync(0xffffffffu, peak_v, o));
      }
      float(&shared)[2][kWarps] = peaks[head & 1];
      if ((threadIdx.x & 31) == 0) {
        shared[0][threadIdx.x >> 5] = peak_k;
        shared[1][threadIdx.x >> 5] = peak_v;
      }
      __syncthreads();                                     // also: every thread has read the old scales
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        peak_k = fmaxf(peak_k, shared[0][w]);
        peak_v = fmaxf(peak_v, shared[1][w]);
      }
      int ek = cache_exponent(peak_k), ev = cache_exponent(peak_v);
      if (first > 0) {                                     // else whatever the page held is no longer there
        ek = max(ek, old_k);
        ev = max(ev, old_v);
      }
      const float sk = power_of_two(-ek), sv = power_of_two(-ev);
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = my_row + i * kRowsAtOnce;
        if (r >= count) continue;
        float vx[kPairs], vy[kPairs];
        rv[i].template values<false>(plain, vx, vy);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          kx[i][j] *= sk;
          ky[i][j] *= sk;
          vx[j] *= sv;
          vy[j] *= sv;
        }
        if ((bad >> i) & 1u) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            kx[i][j] = ky[i][j] = __int_as_float(0x7fffffff);
            vx[j] = vy[j] = 0.0f;
          }
        }
        uint8_t *dk = ck + static_cast<long long>(first + r) * D, *dv = cv + static_cast<long long>(first + r) * D;
        if constexpr (kLanes > 0) {
          if constexpr (kNeighbours) pairs_to_runs(kx[i], ky[i]);
          if (l.live > 0) {
            *reinterpret_cast<uint2*>(dk + l.first[0]) = e4m3_eight(kx[i]);
            *reinterpret_cast<uint2*>(dk + l.second[0]) = e4m3_eight(ky[i]);
            const uint2 lo = e4m3_eight(vx), hi = e4m3_eight(vy);
            *reinterpret_cast<uint4*>(dv + plain.first[0]) = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            if (j < l.live) {
              const uint32_t k2 = e4m3_pair(kx[i][j], ky[i][j]), v2 = e4m3_pair(vx[j], vy[j]);
              dk[l.first[j]] = static_cast<uint8_t>(k2);
              dk[l.second[j]] = static_cast<uint8_t>(k2 >> 8);
              dv[plain.first[j]] = static_cast<uint8_t>(v2);
              dv[plain.second[j]] = static_cast<uint8_t>(v2 >> 8);
            }
          }
        }
      }
      if (head + 1 < head1) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) rv[i].load(v_row[i] += args.v_head, plain);
      }
      if (first > 0) {                                     // the page's older tokens, where the scale has grown
        const int vecs = first * D / 16;
        for (int part = 0; part < 2; ++part) {
          const int grown = part == 0 ? ek - old_k : ev - old_v;
          if (grown == 0) continue;
          uint4* p = reinterpret_cast<uint4*>(part == 0 ? ck : cv);
          const float factor = power_of_two(-min(grown, 126));
          for (int i = threadIdx.x; i < vecs; i += kHeadThreads) {
            const uint4 o = p[i];
            p[i] = make_uint4(e4m3_rescaled(o.x, factor), e4m3_rescaled(o.y, factor), e4m3_rescaled(o.z, factor), e4m3_rescaled(o.w, factor));
          }
        }
      }
      if (threadIdx.x == 0) {
        args.cache.k_scales[block] = static_cast<uint8_t>(ek + 127);
        args.cache.v_scales[block] = static_cast<uint8_t>(ev + 127);
      }
    }
  }

  if (args.q.x == nullptr) return;
  // The queries that go with these heads: the lanes of a row take a few heads of a token in turn, with its rotation in registers.
  const int q0 = head0 * args.group, heads = (head1 - head0) * args.group;
  const int turn_heads = min(8, max(1, heads * count / kRowsAtOnce)), shares = (heads + turn_heads - 1) / turn_heads;
  constexpr int kAhead = kRows > 1 ? 4 : 2;                // small pages and single tokens give a row's lanes few heads
  for (int base = 0; base < count * shares; base += kRowsAtOnce) {
    const int i = base + my_row, share = i % shares, token = i / shares;
    const bool there = token < count;
    const int from_head = share * turn_heads, mine = there ? min(turn_heads, heads - from_head) : 0;
    float wx[kPairs], wy[kPairs];
    head_weights<kNeighbours>(l, args.q.weight != nullptr ? weights[0] : nullptr, wx, wy);
    float c[kPairs], s[kPairs];
    head_turns(l, turns + 2 * (there ? token : 0) * pairs, pairs, c, s);
    const HeadTurn<kPairs> turn(wx, wy, c, s);
    const long long row = row0 + (there ? token : 0);
    const T* const some = static_cast<const T*>(args.q.x) + row * args.q.x_token + q0 * args.q.x_head;
    const T* src = some + from_head * args.q.x_head;
    T* dst = static_cast<T*>(args.q.y) + row * args.q.y_token + (q0 + from_head) * args.q.y_head;
    for (int h = 0; h < turn_heads; h += kAhead) {
      Raw raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u].load(h + u < mine ? src + u * args.q.x_head : some, l);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float x[kPairs], y[kPairs];
        raw[u].template values<kNeighbours>(l, x, y);
        turn.apply(l, args.rot.pairs, x, y, args.norm ? head_norm(l, x, y, inv_columns, args.eps) : 1.0f);
        if (h + u < mine) head_store<kNeighbours>(dst + u * args.q.y_head, l, x, y);
      }
      src += kAhead * args.q.x_head;
      dst += kAhead * args.q.y_head;
    }
  }
}

}  // namespace tb200
