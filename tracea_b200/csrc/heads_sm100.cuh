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
constexpr int kCacheMinExponent = -40, kCacheMaxExponent = 40;

struct Rotation {
  const double* frequencies;   // angle per position of a pair, in radians
  int pairs;                   // 0: no rotation
  int interleaved;             // pair i is columns 2i and 2i + 1; else i and i + pairs
};

// Cosine and sine of position * frequency. The angle is taken in turns and in 64 bits, and so are the quarter turns that are cut
// off: fp32 would be off by 2^-24 of an angle that grows with the position.
__device__ __forceinline__ float2 rotation_of(int position, double frequency) {
  const double quarters = static_cast<double>(position) * frequency * 0.63661977236758134308;   // 2 / pi
  const double whole = rint(quarters);
  const int quadrant = static_cast<int>(static_cast<long long>(whole) & 3);
  float s, c;
  sincospif(0.5f * static_cast<float>(quarters - whole), &s, &c);
  if (quadrant & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  return (quadrant & 2) ? make_float2(-c, -s) : make_float2(c, s);
}

// ------------------------------------------------------------------ a lane's columns of a row
// kVec: 16 columns, lane c of the row in two runs of 8: 8c and 8c + pairs, which a rotation of halves pairs, for the rotated columns
// of that kind; 16c and 16c + 8 for others. Rows are 16-byte aligned, D and the rotated columns multiples of 16.
// Else: kPairs pairs of columns, pair number lane + 32 i, of any row of an even number of columns, which a warp holds.
template <bool kVec, int kScalarPairs>
struct HeadLane {
  static constexpr int kPairs = kVec ? 8 : kScalarPairs;
  int first[kVec ? 1 : kPairs], second[kVec ? 1 : kPairs];   // columns; -1: none
  int angle;                                                 // number of the first pair's angle
  bool live, turned, neighbours;

  __device__ __forceinline__ HeadLane(int lane, int D, const Rotation& rot) {
    neighbours = rot.interleaved != 0;
    if constexpr (kVec) {
      live = 16 * lane < D;
      turned = 16 * lane < 2 * rot.pairs;
      angle = 8 * lane;
      const bool halves = turned && !neighbours;
      first[0] = halves ? 8 * lane : 16 * lane;
      second[0] = halves ? 8 * lane + rot.pairs : 16 * lane + 8;
    } else {
      live = turned = true;
      angle = lane;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int p = lane + 32 * i;
        const bool halves = p < rot.pairs && !neighbours;
        first[i] = 2 * p < D ? (halves ? p : 2 * p) : -1;
        second[i] = halves ? p + rot.pairs : 2 * p + 1;
      }
    }
  }
};

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
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = static_cast<float>(e[i]);
}
// A lane's columns of a row as they lie in memory.
template <typename T, bool kVec, int kScalarPairs>
struct HeadRaw {
  using Lane = HeadLane<kVec, kScalarPairs>;
  Vec8<T> va, vb;
  T sa[kScalarPairs], sb[kScalarPairs];

  __device__ __forceinline__ void load(const T* row, const Lane& l, bool live) {
    if constexpr (kVec) {
      if (live && l.live) {
        fetch8(row + l.first[0], va);
        fetch8(row + l.second[0], vb);
      } else {
        memset(&va, 0, sizeof(va));
        memset(&vb, 0, sizeof(vb));
      }
    } else {
#pragma unroll
      for (int i = 0; i < Lane::kPairs; ++i) {
        const bool here = live && l.first[i] >= 0;
        sa[i] = here ? row[l.first[i]] : static_cast<T>(0.0f);
        sb[i] = here ? row[l.second[i]] : static_cast<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ void values(float (&a)[Lane::kPairs], float (&b)[Lane::kPairs]) const {
    if constexpr (kVec) {
      widen8(va, a);
      widen8(vb, b);
    } else {
#pragma unroll
      for (int i = 0; i < Lane::kPairs; ++i) {
        a[i] = static_cast<float>(sa[i]);
        b[i] = static_cast<float>(sb[i]);
      }
    }
  }
};

// The norm of a row (a mean over D columns; `lanes` lanes, a power of two, hold it) times `weight`, fp32 in shared memory, or nullptr.
template <bool kVec, int kScalarPairs>
__device__ __forceinline__ void head_norm(const HeadLane<kVec, kScalarPairs>& l, float (&a)[HeadLane<kVec, kScalarPairs>::kPairs],
                                          float (&b)[HeadLane<kVec, kScalarPairs>::kPairs], int lanes, float inv_columns, float eps,
                                          const float* weight) {
  constexpr int kPairs = HeadLane<kVec, kScalarPairs>::kPairs;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) sum += a[i] * a[i] + b[i] * b[i];
  for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = 1.0f / sqrtf(sum * inv_columns + eps);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    a[i] *= inv;
    b[i] *= inv;
  }
  if (weight == nullptr) return;
  if constexpr (kVec) {
    if (l.live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] *= weight[l.first[0] + i];
        b[i] *= weight[l.second[0] + i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if (l.first[i] >= 0) {
        a[i] *= weight[l.first[i]];
        b[i] *= weight[l.second[i]];
      }
    }
  }
}

__device__ __forceinline__ void turn_pair(float& a, float& b, float2 cs) {
  const float x = a * cs.x - b * cs.y;
  b = b * cs.x + a * cs.y;
  a = x;
}
// `turns`: the token's cosines and sines, of pair 0 on, in shared memory.
template <bool kVec, int kScalarPairs>
__device__ __forceinline__ void head_turn(const HeadLane<kVec, kScalarPairs>& l, float (&a)[HeadLane<kVec, kScalarPairs>::kPairs],
                                          float (&b)[HeadLane<kVec, kScalarPairs>::kPairs], const float2* turns, int pairs) {
  if constexpr (kVec) {
    if (!l.turned) return;
    float2 cs[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(turns + l.angle + 2 * i);
      cs[2 * i] = make_float2(v.x, v.y);
      cs[2 * i + 1] = make_float2(v.z, v.w);
    }
    if (!l.neighbours) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(a[i], b[i], cs[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn_pair(a[2 * i], a[2 * i + 1], cs[i]);
        turn_pair(b[2 * i], b[2 * i + 1], cs[4 + i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScalarPairs; ++i)
      if (l.angle + 32 * i < pairs) turn_pair(a[i], b[i], turns[l.angle + 32 * i]);
  }
}

template <typename T, bool kVec, int kScalarPairs>
__device__ __forceinline__ void head_store(T* row, const HeadLane<kVec, kScalarPairs>& l,
                                           const float (&a)[HeadLane<kVec, kScalarPairs>::kPairs],
                                           const float (&b)[HeadLane<kVec, kScalarPairs>::kPairs]) {
  if constexpr (kVec) {
    if (l.live) {
      store8(row + l.first[0], a);
      store8(row + l.second[0], b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScalarPairs; ++i) {
      if (l.first[i] >= 0) {
        row[l.first[i]] = static_cast<T>(a[i]);
        row[l.second[i]] = static_cast<T>(b[i]);
      }
    }
  }
}

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
  int lanes;                   // lanes of a row
  int splits, passes;          // warps of a token; passes of a warp over 32 / lanes heads that a token takes in all
  float eps;
};

template <typename T>
__device__ __forceinline__ void weights_to_shared(float* dst, const void* weight, int is_f32, int D) {
  if (weight == nullptr) return;
  for (int i = threadIdx.x; i < D; i += kHeadThreads)
    dst[i] = is_f32 ? static_cast<const float*>(weight)[i] : static_cast<float>(static_cast<const T*>(weight)[i]);
}

// A warp takes a token's heads 32 / lanes at a time, or, where the tokens alone would not fill the machine, a share of them. Two
// passes' loads are under way at once.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kHeadThreads) head_rotate_kernel(const __grid_constant__ HeadRotateArgs args) {
  using Lane = HeadLane<kVec, 4>;
  constexpr int kPairs = Lane::kPairs, kAhead = 2;
  __shared__ float weights[2][kHeadMaxColumns];
  __shared__ __align__(16) float2 turns[kHeadThreads / 32][kHeadMaxColumns / 2];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long id = static_cast<long long>(blockIdx.x) * (kHeadThreads / 32) + warp;
  const int token = static_cast<int>(id / args.splits), split = static_cast<int>(id % args.splits);
  for (int r = 0; r < 2; ++r) weights_to_shared<T>(weights[r], args.rows[r].weight, args.rows[r].weight_f32, args.D);
  if (token < args.tokens && args.rot.pairs > 0) {
    const int position = args.positions[token];
    for (int p = lane; p < args.rot.pairs; p += 32) turns[warp][p] = rotation_of(position, args.rot.frequencies[p]);
  }
  __syncthreads();
  if (token >= args.tokens) return;
  const int lanes = kVec ? args.lanes : 32, group = lane / lanes, per_pass = 32 / lanes;
  const Lane l(lane % lanes, args.D, args.rot);
  const int heads = args.rows[0].heads + args.rows[1].heads;
  const int begin = static_cast<int>(static_cast<long long>(args.passes) * split / args.splits);
  const int end = static_cast<int>(static_cast<long long>(args.passes) * (split + 1) / args.splits);
  const float inv_columns = 1.0f / static_cast<float>(args.D);
  for (int pass = begin; pass < end; pass += kAhead) {
    HeadRaw<T, kVec, 4> raw[kAhead];
    int head[kAhead], which[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      head[u] = (pass + u) * per_pass + group;
      const bool live = pass + u < end && head[u] < heads;
      which[u] = head[u] >= args.rows[0].heads ? 1 : 0;
      if (which[u]) head[u] -= args.rows[0].heads;
      if (!live) head[u] = -1;
      const HeadRows& rows = args.rows[which[u]];
      raw[u].load(static_cast<const T*>(rows.x) + token * rows.x_token + (live ? head[u] : 0) * rows.x_head, l, live);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float a[kPairs], b[kPairs];
      raw[u].values(a, b);
      const HeadRows& rows = args.rows[which[u]];
      if (args.norm) head_norm(l, a, b, lanes, inv_columns, args.eps, rows.weight != nullptr ? weights[which[u]] : nullptr);
      head_turn(l, a, b, turns[warp], args.rot.pairs);
      if (head[u] >= 0) head_store(static_cast<T*>(rows.y) + token * rows.y_token + head[u] * rows.y_head, l, a, b);
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
__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) { return e4m3_pair(a, b) | (e4m3_pair(c, d) << 16); }
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
  int norm, lanes;
  int group;                   // heads of q to one of k
  int heads_per_cta;           // of k
  int turn_rows;               // rows of angles in shared memory
  float eps;
};

// A CTA takes the new tokens of one page of a sequence, and some heads: for each the keys and values, whose scales need all of the
// block's rows and so stay in registers until they are known, and the queries' heads that go with it. A block belongs to one CTA:
// nothing is shared, nothing atomic. kRows: rows of a block that a lane holds.
template <typename T, bool kVec, int kRows>
__global__ void __launch_bounds__(kHeadThreads) kv_append_kernel(const __grid_constant__ KvAppendArgs args) {
  constexpr int kScalarPairs = kCacheMaxColumns / 64;
  using Lane = HeadLane<kVec, kScalarPairs>;
  constexpr int kPairs = Lane::kPairs, kWarps = kHeadThreads / 32;
  extern __shared__ __align__(16) float2 turns[];          // [turn_rows][pairs]
  __shared__ float weights[2][kCacheMaxColumns];
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
  long long page = -1;
  if (slot >= 0 && slot < args.seqs.table_width) page = args.seqs.table[at.sequence * args.seqs.table_stride + slot];
  if (page >= args.cache.pages) page = -1;

  weights_to_shared<T>(weights[0], args.q.weight, args.q.weight_f32, D);
  weights_to_shared<T>(weights[1], args.k.weight, args.k.weight_f32, D);
  const int pairs = args.rot.pairs;
  for (int i = threadIdx.x; i < count * pairs; i += kHeadThreads) {
    const int r = i / pairs, p = i - r * pairs;
    turns[i] = rotation_of(from + r, args.rot.frequencies[p]);
  }
  __syncthreads();

  const int lanes = kVec ? args.lanes : 32, rows_at_once = kHeadThreads / lanes;
  const int my_row = static_cast<int>(threadIdx.x) / lanes, my_lane = static_cast<int>(threadIdx.x) % lanes;
  const Lane l(my_lane, D, args.rot);
  const Lane plain(my_lane, D, Rotation{nullptr, 0, 0});   // values are not rotated: their columns in order
  const float inv_columns = 1.0f / static_cast<float>(D);
  const int head0 = static_cast<int>(blockIdx.y) * args.heads_per_cta, head1 = min(args.cache.heads, head0 + args.heads_per_cta);

  if (page >= 0) {
    for (int head = head0; head < head1; ++head) {
      const long long block = page * args.cache.heads + head;
      uint8_t* ck = args.cache.k + (block << shift) * D;
      uint8_t* cv = args.cache.v + (block << shift) * D;
      const int old_k = static_cast<int>(args.cache.k_scales[block]) - 127, old_v = static_cast<int>(args.cache.v_scales[block]) - 127;
      HeadRaw<T, kVec, kScalarPairs> rk[kRows], rv[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = my_row + i * rows_at_once;
        const long long row = row0 + r;
        rk[i].load(static_cast<const T*>(args.k.x) + row * args.k.x_token + head * args.k.x_head, l, r < count);
        rv[i].load(static_cast<const T*>(args.v) + row * args.v_token + head * args.v_head, plain, r < count);
      }
      float ka[kRows][kPairs], kb[kRows][kPairs];
      float peak_k = 0.0f, peak_v = 0.0f;
      uint32_t bad = 0u;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        rk[i].values(ka[i], kb[i]);
        if (args.norm) head_norm(l, ka[i], kb[i], lanes, inv_columns, args.eps, args.k.weight != nullptr ? weights[1] : nullptr);
        if (my_row + i * rows_at_once < count) head_turn(l, ka[i], kb[i], turns + (my_row + i * rows_at_once) * pairs, pairs);
        float va[kPairs], vb[kPairs];
        rv[i].values(va, vb);
        float mk = 0.0f, mv = 0.0f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          mk = fmaxf(mk, fmaxf(fabsf(ka[i][j]), fabsf(kb[i][j])));
          mv = fmaxf(mv, fmaxf(fabsf(va[j]), fabsf(vb[j])));
          finite = finite && isfinite(ka[i][j]) && isfinite(kb[i][j]) && isfinite(va[j]) && isfinite(vb[j]);
        }
        // a token that is not finite counts for no scale: a vote of its lanes
        const uint32_t votes = __ballot_sync(0xffffffffu, !finite);
        const uint32_t mine = lanes == 32 ? votes : (votes >> ((threadIdx.x & 31) / lanes * lanes)) & ((1u << lanes) - 1u);
        if (mine != 0u) bad |= 1u << i;
        else {
          peak_k = fmaxf(peak_k, mk);
          peak_v = fmaxf(peak_v, mv);
        }
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
        const int r = my_row + i * rows_at_once;
        if (r >= count) continue;
        const bool drop = (bad >> i) & 1u;
        float va[kPairs], vb[kPairs];
        rv[i].values(va, vb);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          ka[i][j] = drop ? __int_as_float(0x7fffffff) : ka[i][j] * sk;
          kb[i][j] = drop ? __int_as_float(0x7fffffff) : kb[i][j] * sk;
          va[j] = drop ? 0.0f : va[j] * sv;
          vb[j] = drop ? 0.0f : vb[j] * sv;
        }
        uint8_t *dk = ck + static_cast<long long>(first + r) * D, *dv = cv + static_cast<long long>(first + r) * D;
        if constexpr (kVec) {
          if (l.live) {
            *reinterpret_cast<uint2*>(dk + l.first[0]) =
                make_uint2(e4m3_four(ka[i][0], ka[i][1], ka[i][2], ka[i][3]), e4m3_four(ka[i][4], ka[i][5], ka[i][6], ka[i][7]));
            *reinterpret_cast<uint2*>(dk + l.second[0]) =
                make_uint2(e4m3_four(kb[i][0], kb[i][1], kb[i][2], kb[i][3]), e4m3_four(kb[i][4], kb[i][5], kb[i][6], kb[i][7]));
            *reinterpret_cast<uint4*>(dv + plain.first[0]) =
                make_uint4(e4m3_four(va[0], va[1], va[2], va[3]), e4m3_four(va[4], va[5], va[6], va[7]),
                           e4m3_four(vb[0], vb[1], vb[2], vb[3]), e4m3_four(vb[4], vb[5], vb[6], vb[7]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            if (l.first[j] >= 0) {
              const uint32_t ek2 = e4m3_pair(ka[i][j], kb[i][j]), ev2 = e4m3_pair(va[j], vb[j]);
              dk[l.first[j]] = static_cast<uint8_t>(ek2);
              dk[l.second[j]] = static_cast<uint8_t>(ek2 >> 8);
              dv[plain.first[j]] = static_cast<uint8_t>(ev2);
              dv[plain.second[j]] = static_cast<uint8_t>(ev2 >> 8);
            }
          }
        }
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
  // the queries that go with these heads
  const int q0 = head0 * args.group, heads = (head1 - head0) * args.group, total = count * heads;
  constexpr int kAhead = 2;
  for (int base = 0; base < total; base += kAhead * rows_at_once) {
    HeadRaw<T, kVec, kScalarPairs> raw[kAhead];
    int token[kAhead], head[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = base + u * rows_at_once + my_row;
      const bool live = i < total;
      token[u] = live ? i / heads : -1;
      head[u] = live ? q0 + i - token[u] * heads : 0;
      raw[u].load(static_cast<const T*>(args.q.x) + (live ? row0 + token[u] : row0) * args.q.x_token + head[u] * args.q.x_head, l, live);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float a[kPairs], b[kPairs];
      raw[u].values(a, b);
      if (args.norm) head_norm(l, a, b, lanes, inv_columns, args.eps, args.q.weight != nullptr ? weights[0] : nullptr);
      if (token[u] >= 0) {
        head_turn(l, a, b, turns + token[u] * pairs, pairs);
        head_store(static_cast<T*>(args.q.y) + (row0 + token[u]) * args.q.y_token + head[u] * args.q.y_head, l, a, b);
      }
    }
  }
}

}  // namespace tb200
