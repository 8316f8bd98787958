// Attention over packed sequences of different lengths, grouped heads, optionally causal.
//
//   o[i, h] = sum_j p_ij v[j, h / G] / sum_j p_ij,   p_ij = exp(scale q[i, h] . k[j, h / G] - m_i)
//
// over the keys j that query i of its sequence sees: all of them, or with `causal` those up to
// i + (keys - queries), so that the last query sees every key whatever the cache holds before the
// first one.  A query that sees no key gives zeros.
//
// A sequence's queries and the G heads that share a key head are one list of rows, token-major:
// row r is token r / G, head r % G of the group.  So the rows of a tile share their keys whatever G
// is, and a single new token still fills G rows of a matrix instruction.
//
// The keys are rows of one tensor (packed sequences, caches of a fixed capacity: sf_packed_attention_args, A below) or
// of pages that a table names (sf_paged_attention_args, PagedArgs).
//
// Two kernels over those rows, joined by a third where the keys are split:
//   packed_tile_kernel    workgroups of many rows: K and V tiles of 64 keys shared through LDS
//   packed_stream_kernel  32 rows: each wave streams its own slice of the keys
//   packed_combine_kernel joins the slices of different workgroups
// and one that counts row tiles before them where there are many sequences (packed_starts_kernel).
#pragma once

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "index.h"
#include "sf_common.h"

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef short v4i16p __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16p lds_v4i16p;

// 16-bit element types: the matrix product, rounding of two weights to one word, their sum.
struct Bf16 {
  // A lane's weights of a tile that sum to more than 2^kMass against the row's reference point move it.  (2^12 moves it more
  // often: prompt of 4096, 32 / 8 heads of 128, logits of deviation 12, 170 us.)
  static constexpr int kMass = 24;
  // All weights of a row are 2^-shift of what the reference point makes them, so that those of n keys together, two
  // lanes of up to 2^kMass each in at most ceil(n / 32) tiles, sum to 1/2 at most: values up to the largest bf16 do not
  // pass fp32 in any partial sum.  (Values below 2^-126 + shift may lose digits instead.)
  static __device__ __forceinline__ float shift(int n) { return (float)(kMass - 3 + max(32 - __clz(n), 5)); }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return __builtin_bit_cast(uint32_t, cvt_bf2(lo, hi)); }
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) { return add_bf2(__builtin_bit_cast(bf16x2, w), acc); }
  static __device__ __forceinline__ float to_float(uint16_t v) { return bf2f(v); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return f2bf(v); }
};
struct Fp16 {
  // Weights of 2^4 at the reference point, finite where a lane's sum to no more than 2^16 (an infinite one does not), and
  // rounded to a multiple of 2^-24: only those below 2^-29 of the reference point's vanish.  (Values are too small to pass
  // fp32.)
  static constexpr int kMass = 12;
  static __device__ __forceinline__ float shift(int) { return -4.f; }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
  }
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) {
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), one, acc, false);
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// A reference point m of a row's products s = q.k: weights are 2^(c (s - m) - shift) with c = |scale| log2 e, one fma and
// one exp2 as 2^(c s - mc), mc = c m + shift.  The rounding of mc scales all weights of the row alike, by up to 2^(1/2)
// while |mc| < 2^24.  Beyond it could be any factor: there mc is NaN, which accepts no tile as it stands, and
// settle() forms the weights from s - m, whose rounding is relative to what it is.  (m = -FLT_MAX: no key yet.)
constexpr float kFar = 0x1p24f;
__device__ __forceinline__ float times(float m, float c) {
  float x = m * c;
  asm("" : "+v"(x));                                         // (rounded here, not within a later fma)
  return x;
}
__device__ __forceinline__ float reference(float m, float c, float shift) {
  const float x = times(m, c) + shift;
  return fabsf(x) < kFar ? x : __builtin_nanf("");
}
// What sums against each of m are worth against mnew, no smaller than any of them.  A difference of the rounded c m
// where none is far, or one lies so far below that it is worth nothing (no key yet).
template <int N>
__device__ __forceinline__ void rescale(const float (&m)[N], float mnew, float c, float shift, float (&w)[N]) {
  const float b = times(mnew, c) + shift;
  float far = fabsf(b);
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const float a = times(m[x], c) + shift;
    far = fmaxf(far, a > -2.f * kFar ? fabsf(a) : 0.f);
    w[x] = a - b;
  }
  if (__any(!(far < kFar))) {
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const float a = times(m[x], c) + shift;
      const float from_far = fabsf(b) < kFar ? __builtin_fmaf(m[x], c, -b) + shift : (m[x] - mnew) * c;
      const float from_near = fabsf(b) < kFar ? w[x] : -(__builtin_fmaf(mnew, c, -a) + shift);
      w[x] = fabsf(a) < kFar ? from_near : from_far;
    }
  }
#pragma unroll
  for (int x = 0; x < N; ++x) w[x] = fast_exp2(w[x]);
}

// Where a cache's rows are.  A page holds a multiple of 16 rows; units of 16 consecutive keys have one page each.
struct PagedArgs : sf_paged_attention_args {
  PageDiv div;                                               // of a page's units (units < 2^27)
};

// A launch dimension holds less than 2^32 threads: workgroups past kGridX (of up to 512) continue in the next row of the grid.
constexpr int kGridX = 1 << 22;
__device__ __forceinline__ int workgroup() { return (int)(blockIdx.y * kGridX + blockIdx.x); }

struct PackedPlan {
  int tiles;         // bound on the row tiles of one key head
  int slices;        // packed_tile_kernel: key slices (workgroups) of every row tile
  int share;         // packed_stream_kernel: slices of all row tiles of a key head together, dealt out by their keys (0: one each)
  int whole;         // with a share: no slices where the longest sequence is near the mean
  int pieces;        // blocks of packed_combine_kernel per row tile
  float c0;          // scale log2 e
  int G;             // query heads of a key head
  double inv_g;      // 1 / G
  float* part;       // of split tiles, per (slice, key head) unnormalised O [R][DP], then (m, l) [R][2]
  int4* found;       // per tile, for the join: (q0, lq, lk, tile of the sequence), (k0, its first slice, slices, -); lq = 0: none
  int* starts;       // more than kScanned sequences: the tiles before each, from packed_starts_kernel; else null
};

// Up to as many sequences every workgroup counts the tiles itself, 64 sequences a step; above, one workgroup
// counts them for all, a launch of its own (sequences of 20 tokens, 8 heads of 64, counted by each / for all: 130 of
// them 20.8 / 22.7 us, 256 37.7 / 31.2, 512 90 / 55, 8192 12370 / 797).
constexpr int kScanned = 192;

// Up to as many share key slices (find_slice).
constexpr int kShared = 256;

// r / G without a division: (r + 0.5) / G is at least 0.5 / G away from a whole number.
__device__ __forceinline__ int token_of(const PackedPlan& pl, int r) { return (int)(((double)r + 0.5) * pl.inv_g); }

// Tile sizes.  KC: 16-dim steps of q.k that hold data; DP: head dim padded to whole 32-dim blocks.
template <int KC>
struct Dims {
  static constexpr int DB = (KC + 1) / 2;                   // 32-dim blocks
  static constexpr int DP = 32 * DB;
  static constexpr int kRow = DP * 2;                       // bytes of a K or V row in LDS
  static constexpr int kPieces = DP / 8;                    // 16-byte pieces of it
  // K: pieces of a row are XORed by key so that the reads of 16 consecutive keys (one piece each) fall
  // on 16 different 16-byte slots of the 256 bytes that the banks span.
  static __device__ __forceinline__ int kpiece(int key, int piece) {
    return DP == 128 ? piece ^ (key & 15) : DP == 64 ? piece ^ ((key >> 1) & 7) : piece ^ ((key >> 2) & 3);
  }
  // V: a transposing read takes 64 bytes of each of 4 consecutive keys: those 64-byte units fall on
  // different quarters of the banks (rows of 64 and 192 bytes do so by themselves).
  static __device__ __forceinline__ int vpiece(int key, int piece) {
    return DP == 128 ? piece ^ ((key & 3) << 2) : DP == 64 ? piece ^ (((key >> 1) & 1) << 2) : piece;
  }
};

// One sequence's part of the operands, clamped to what the tensors hold whatever the offsets say.
struct Seq {
  int q0, lq, k0, lk;
};
__device__ __forceinline__ void seq_range(const int32_t* cu, const int32_t* len, int b, int64_t total, int& start, int& n) {
  const int64_t s = min(max((int64_t)cu[b], (int64_t)0), total);
  int64_t e = min(max((int64_t)cu[b + 1], s), total);
  if (len != nullptr) e = min(e, s + max(len[b], 0));
  start = (int)s;
  n = (int)(e - s);
}

__device__ __forceinline__ void key_range(const sf_packed_attention_args& a, int b, int& k0, int& lk) {
  seq_range(a.cu_k, a.len_k, b, a.Tk, k0, lk);
}
// (of a paged cache, k0 is the sequence: its row of the table)
__device__ __forceinline__ void key_range(const PagedArgs& a, int b, int& k0, int& lk) {
  k0 = b;
  lk = (int)min((int64_t)max(a.len_k[b], 0), (int64_t)a.table_cols * a.page_rows);
}

// Row 0 of what a page that does not exist holds.
__device__ const u32x4 kZeros[16] = {};

// Rows of keys and values of one sequence and key head, one by one.
template <class A>
struct KeyRows;
template <>
struct KeyRows<sf_packed_attention_args> {
  const uint16_t *kp, *vp;
  int64_t ks, vs;
  __device__ __forceinline__ KeyRows(const sf_packed_attention_args& a, const Seq& s, int hk)
      : kp((const uint16_t*)a.k + (int64_t)s.k0 * a.k_s[0] + (int64_t)hk * a.k_s[1]),
        vp((const uint16_t*)a.v + (int64_t)s.k0 * a.v_s[0] + (int64_t)hk * a.v_s[1]), ks(a.k_s[0]), vs(a.v_s[0]) {}
  __device__ __forceinline__ const uint16_t* k(int j) const { return kp + (int64_t)j * ks; }
  __device__ __forceinline__ const uint16_t* v(int j) const { return vp + (int64_t)j * vs; }
};
template <>
struct KeyRows<PagedArgs> {
  const PagedArgs& a;
  const int32_t* table;
  int head;
  __device__ __forceinline__ KeyRows(const PagedArgs& args, const Seq& s, int hk)
      : a(args), table(args.table + s.k0 * args.table_s), head(hk) {}
  __device__ __forceinline__ const uint16_t* row(const void* p, const int64_t (&st)[3], int j) const {
    const int page = j / a.page_rows, id = table[page];
    if ((uint32_t)id >= (uint32_t)a.pages) return reinterpret_cast<const uint16_t*>(kZeros);
    return (const uint16_t*)p + id * st[0] + (j - page * a.page_rows) * st[1] + head * st[2];
  }
  __device__ __forceinline__ const uint16_t* k(int j) const { return row(a.k, a.k_s, j); }
  __device__ __forceinline__ const uint16_t* v(int j) const { return row(a.v, a.v_s, j); }
};

// Sums of int or float over lanes 0 .. own, and over all; every lane calls.  Rows of 16 lanes by shifts, then the rows.
template <class V>
__device__ __forceinline__ V row_sums(V v) {
  v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x111, 0xF, 0xF, false));   // row_shr 1, 2, 4, 8
  v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x112, 0xF, 0xF, false));
  v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x114, 0xF, 0xF, false));
  v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x118, 0xF, 0xF, false));
  return v;
}
template <class V>
__device__ __forceinline__ V row_sum(V v, int lane) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ int lanes_before_and_own(int v) {
  const int lane = threadIdx.x & 63;
  v = row_sums(v);
  const int r0 = row_sum(v, 15), r1 = r0 + row_sum(v, 31), r2 = r1 + row_sum(v, 47);
  return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}
template <class V>
__device__ __forceinline__ V lanes_sum(V v) {
  v = row_sums(v);
  return (row_sum(v, 15) + row_sum(v, 31)) + (row_sum(v, 47) + row_sum(v, 63));
}

// Tile `idx` of the sequences' row tiles of R rows each, laid end to end: its sequence and its index
// there, or false past the last.  All lanes of the wave take part; the results are uniform.
template <int R, class A>
__device__ __forceinline__ bool find_tile(const A& a, const PackedPlan& pl, int idx, Seq& s, int& tile, int& ntiles) {
  const int lane = threadIdx.x & 63;
  if (pl.starts != nullptr) {
    if (idx >= pl.starts[a.B]) return false;
    // the last sequence that starts at or before idx, among n from b on: 64 of them a step
    int b = 0, n = a.B;
    while (n > 1) {
      const int step = (n + 63) / 64;
      const bool at = lane * step < n && pl.starts[b + min(lane * step, n - 1)] <= idx;
      const int skip = max(__popcll(__ballot(at)) - 1, 0) * step;
      b += skip;
      n = min(step, n - skip);
    }
    seq_range(a.cu_q, a.len_q, b, a.Tq, s.q0, s.lq);
    key_range(a, b, s.k0, s.lk);
    ntiles = (int)(((uint32_t)s.lq * (uint32_t)pl.G + R - 1) / R);
    tile = idx - pl.starts[b];
    return tile < ntiles;
  }
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int start = 0, n = 0, k0 = 0, lk = 0;
    if (b < a.B) {
      seq_range(a.cu_q, a.len_q, b, a.Tq, start, n);
      key_range(a, b, k0, lk);
    }
    const int nt = (int)(((uint32_t)n * (uint32_t)pl.G + R - 1) / R);      // (rows fit 31 bits)
    const int incl = lanes_before_and_own(nt);
    const uint64_t past = __ballot(base + incl > idx);
    if (past != 0) {
      const int src = __builtin_ctzll(past);
      s.q0 = __builtin_amdgcn_readlane(start, src);
      s.lq = __builtin_amdgcn_readlane(n, src);
      s.k0 = __builtin_amdgcn_readlane(k0, src);
      s.lk = __builtin_amdgcn_readlane(lk, src);
      ntiles = __builtin_amdgcn_readlane(nt, src);
      tile = idx - base - (__builtin_amdgcn_readlane(incl, src) - ntiles);
      return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// The tile that is number `idx` of all by the keys that it sees, most first (in steps of 64), or false past the
// last: up to 64 sequences, a lane each.  The steps u of 64 keys are searched for the one where more
// than idx tiles see more than 64 u keys, but not 64 (u + 1).
template <int R, class A>
__device__ __forceinline__ bool find_longest(const A& a, const PackedPlan& pl, int idx, Seq& s, int& tile) {
  const int lane = threadIdx.x & 63;
  int start = 0, n = 0, k0 = 0, lk = 0;
  if (lane < a.B) {
    seq_range(a.cu_q, a.len_q, lane, a.Tq, start, n);
    key_range(a, lane, k0, lk);
  }
  const int nt = (int)(((uint32_t)n * (uint32_t)pl.G + R - 1) / R);
  const auto longer = [&](int u) __attribute__((always_inline)) {              // of the lane's sequence
    if (u < 0) return nt;
    if (!a.causal) return lk > 64 * u ? nt : 0;
    const int token = 64 * u - (lk - n);                     // the first that sees more than 64 u keys
    return token <= 0 ? nt : token >= n ? 0 : nt - (int)((uint32_t)token * (uint32_t)pl.G / R);
  };
  if (lanes_sum(nt) <= idx) return false;
  int step = 1, u = -1;
  while (__any(lk > 64 * step) && step < 1 << 24) step <<= 1;
  for (; step > 0; step >>= 1)
    if (lanes_sum(longer(u + step)) > idx) u += step;
  const int above = longer(u + 1), here = longer(u) - above, rank = idx - lanes_sum(above);
  const int incl = lanes_before_and_own(here);
  const uint64_t past = __ballot(incl > rank);
  if (past == 0) return false;                               // (not with offsets that increase)
  const int src = __builtin_ctzll(past);
  s.q0 = __builtin_amdgcn_readlane(start, src);
  s.lq = __builtin_amdgcn_readlane(n, src);
  s.k0 = __builtin_amdgcn_readlane(k0, src);
  s.lk = __builtin_amdgcn_readlane(lk, src);
  const int ntiles = __builtin_amdgcn_readlane(nt, src);
  tile = ntiles - 1 - __builtin_amdgcn_readlane(above, src) - (rank - __builtin_amdgcn_readlane(incl - here, src));
  return tile >= 0 && tile < ntiles;
}

// starts[b]: row tiles of the sequences before b, starts[B] those of all.  One workgroup.
template <class A>
__global__ __launch_bounds__(1024) void packed_starts_kernel(const A a, const PackedPlan pl, int R) {
  constexpr int kEach = 4;
  __shared__ int64_t waves[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t base = 0;                                          // (offsets that overlap may count more than 31 bits hold)
  for (int64_t b0 = 0; b0 < a.B; b0 += 1024 * kEach) {
    const int64_t b = b0 + kEach * threadIdx.x;
    int64_t nt[kEach], sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      int start, n = 0;
      if (b + e < a.B) seq_range(a.cu_q, a.len_q, (int)(b + e), a.Tq, start, n);
      nt[e] = ((uint32_t)n * (uint32_t)pl.G + R - 1) / R;
      sum += nt[e];
    }
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = __shfl_up((long long)incl, o);
      incl += lane >= o ? up : 0;
    }
    if (lane == 63) waves[wave] = incl;
    __syncthreads();
    int64_t before = base + incl - sum;
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? waves[w] : 0;
      base += waves[w];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (b + e < a.B) pl.starts[b + e] = (int)min(before, (int64_t)INT32_MAX);
      before += nt[e];
    }
  }
  if (threadIdx.x == 0) pl.starts[a.B] = (int)min(base, (int64_t)INT32_MAX);
}

// Leaves to packed_combine_kernel what tile `slot` is.
__device__ __forceinline__ void note_tile(const PackedPlan& pl, int slot, bool there, const Seq& s, int tile, int first, int slices) {
  pl.found[2 * slot] = there ? int4{s.q0, s.lq, s.lk, tile} : int4{0, 0, 0, 0};
  pl.found[2 * slot + 1] = there ? int4{s.k0, first, slices, 0} : int4{0, 0, 0, 0};
}

// Whether packed_tile_kernel's slices may be dealt out by the keys too (its rule is in route()).
template <class A>
constexpr bool kShareTiles = std::is_same<A, PagedArgs>::value;

// Slice `item` of all, where the tiles of up to 64 N sequences (N a lane) share pl.share slices by their keys, in
// slices of c units of `unit` keys: the smallest c that needs no more than the share, one slice a tile aside.  c is at
// least all units / share, which needs share + tiles at most (the launch's bound), and at most all units / (share - tiles).
// False past the last; `slot` is the tile's number among all, past the last slice one that no tile has.
template <int R, int N, class A>
__device__ __forceinline__ bool find_slice(const A& a, const PackedPlan& pl, int unit, int item, Seq& s, int& tile,
                                           int& slot, int& slice, int& slices) {
  const int lane = threadIdx.x & 63;
  int start[N], n[N], k0[N], lk[N], nt[N], units[N], own_tiles = 0, longest = 0;
  float own_units = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int b = N * lane + j;
    start[j] = n[j] = k0[j] = lk[j] = 0;
    if (b < a.B) {
      seq_range(a.cu_q, a.len_q, b, a.Tq, start[j], n[j]);
      key_range(a, b, k0[j], lk[j]);
    }
    nt[j] = (int)(((uint32_t)n[j] * (uint32_t)pl.G + R - 1) / R);
    units[j] = (lk[j] + unit - 1) / unit;
    own_tiles += nt[j];
    own_units += (float)nt[j] * (float)units[j];
    longest = max(longest, units[j]);
  }
  const int tiles = lanes_before_and_own(own_tiles), all = __builtin_amdgcn_readlane(tiles, 63);
  slot = item;
  if (all > pl.tiles) return false;                          // (offsets that do not increase)
  const float total = lanes_sum(own_units);
  const auto over = [&](int n) __attribute__((always_inline)) {                // ceil(total / n)
    // (whole numbers up to 2^23 are exact; above, the quotient is kept from falling short)
    return total < 8388608.f ? max(((uint32_t)total + n - 1) / n, 1u) : (uint32_t)fminf(ceilf(total / (float)n * 1.000001f), 1e9f);
  };
  const auto split = [&](int j, uint32_t c) __attribute__((always_inline)) { return (int)max((units[j] + c - 1) / c, 1u); };
  const auto needs = [&](uint32_t c) __attribute__((always_inline)) {          // the lane's slices
    int v = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) v += nt[j] * split(j, c);
    return v;
  };
  uint32_t c = over(pl.share);
  if (pl.whole && !__any((float)longest * (float)all > 1.25f * total)) c = 1u << 30;
  const bool fits = pl.share <= all || c == 1u << 30 || lanes_sum(needs(c)) <= pl.share;
  for (uint32_t high = fits ? c : over(pl.share - all); c < high;) {
    const uint32_t mid = (c + high) / 2;
    if (lanes_sum(needs(mid)) <= pl.share) high = mid;
    else c = mid + 1;
  }
  const int own_items = needs(c), items = lanes_before_and_own(own_items);
  const uint64_t past = __ballot(items > item);
  if (past == 0) {
    slot = all + item - __builtin_amdgcn_readlane(items, 63);
    return false;
  }
  const int src = __builtin_ctzll(past);
  int r = item - __builtin_amdgcn_readlane(items - own_items, src);
  slot = __builtin_amdgcn_readlane(tiles - own_tiles, src);
  bool found = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int ntj = __builtin_amdgcn_readlane(nt[j], src), z = __builtin_amdgcn_readlane(split(j, c), src);
    if (!found && r < ntj * z) {
      found = true;
      s.q0 = __builtin_amdgcn_readlane(start[j], src);
      s.lq = __builtin_amdgcn_readlane(n[j], src);
      s.k0 = __builtin_amdgcn_readlane(k0[j], src);
      s.lk = __builtin_amdgcn_readlane(lk[j], src);
      slices = z;
    } else if (!found) {
      r -= ntj * z;
      slot += ntj;
    }
  }
  tile = r / slices;
  slice = r - tile * slices;
  slot += tile;
  return true;
}

// Last key that row r of the sequence sees (-1: none).
__device__ __forceinline__ int last_key(const Seq& s, int causal, int r, const PackedPlan& pl) {
  return causal ? max(min(token_of(pl, r) + s.lk - s.lq, s.lk - 1), -1) : s.lk - 1;
}

// Element offset of row r in q or out: token, head.
__device__ __forceinline__ int64_t row_at(const Seq& s, const PackedPlan& pl, int hk, int r, const int64_t (&stride)[2]) {
  const int token = token_of(pl, r);
  return (int64_t)(s.q0 + token) * stride[0] + (int64_t)(hk * pl.G + r - token * pl.G) * stride[1];
}

// Offset of pieces that do not exist.  A tile's last byte lies below it (row strides below 2^25 bytes, 64
// rows), and so does what the rows' steps add to it below 2^32.
constexpr uint32_t kOutside = 0x80000000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int64_t bytes) {
  // raw buffer, 32-bit data: loads past `bytes` return zeros
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// What a wave holds of its 32 rows: lane (li, half) has row li; o[db][r] is dim 32 db + 8 (r / 4) +
// 4 half + r % 4; l is the lane's own part of the sum (its keys).
template <class E, int KC>
struct RowState {
  using T = Dims<KC>;
  u32x4 q[KC];                                               // Q operand: dims 16 kk + 8 half .. +7
  f32x16 o[T::DB];
  float m, l, c0, mc, shift, limit;                          // mc: reference(m, c0, shift); limit: 2^(E::kMass - shift)

  template <class A>
  __device__ __forceinline__ void init(const A& a, const PackedPlan& pl, const Seq& s, int r, int hk) {
    const int half = (threadIdx.x >> 5) & 1;
    const uint16_t* qp = (const uint16_t*)a.q + row_at(s, pl, hk, r, a.q_s);
#pragma unroll
    for (int kk = 0; kk < KC; ++kk) {
      const int d0 = 16 * kk + 8 * half;
      q[kk] = d0 < a.D ? ld16(qp + d0) : u32x4{0, 0, 0, 0};
    }
    // a negative scale turns the queries over, so that the largest product has the largest logit
    if (pl.c0 < 0.f)
#pragma unroll
      for (int kk = 0; kk < KC; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) q[kk][e] ^= 0x80008000u;
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[db][x] = 0.f;
    m = -FLT_MAX;
    l = 0.f;
    c0 = fabsf(pl.c0);
    asm("" : "+v"(c0));                                      // (an fma that takes it from a scalar register issues more slowly)
    shift = E::shift(s.lk);
    limit = __uint_as_float((uint32_t)(127 + E::kMass - (int)shift) << 23);
    mc = reference(m, c0, shift);
  }

  // S^T = K Q^T of a tile of 32 NB keys in LDS: lane (row li) gets keys 32 kb + 8 (r / 4) + 4 half + r % 4.
  // The operands are read kAhead products before they are taken; `between(x)` is issued after product x.
  template <int NB, class F>
  __device__ __forceinline__ void products(const uint8_t* kt, f32x16 (&s)[NB], F between) const {
    const int half = (threadIdx.x >> 5) & 1, li = threadIdx.x & 31;
    constexpr int kAll = NB * KC, kAhead = kAll < 4 ? kAll : 4;
    const auto operand = [&](int x) __attribute__((always_inline)) {
      const int key = 32 * (x % NB) + li;
      return ld16(kt + key * T::kRow + (T::kpiece(key, 2 * (x / NB) + half) << 4));
    };
    u32x4 k[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) k[x] = operand(x);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int x = 0; x < 16; ++x) s[kb][x] = 0.f;
#pragma unroll
    for (int x = 0; x < kAll; ++x) {
      s[x % NB] = E::mfma(k[x % kAhead], q[x / NB], s[x % NB]);
      if (x + kAhead < kAll) k[x % kAhead] = operand(x + kAhead);
      between(x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Weight 0 for the keys past `last`, of the tile.
  template <int NB>
  __device__ __forceinline__ void hide(f32x16 (&s)[NB], int last) const {
    last -= 4 * ((threadIdx.x >> 5) & 1);                    // (so that the keys are constants)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int x = 0; x < 16; ++x) s[kb][x] = 32 * kb + 8 * (x >> 2) + (x & 3) > last ? -INFINITY : s[kb][x];
  }

  // Weights against a reference point that stays where an earlier tile put it, until a tile's weights
  // sum to more than the limit (or to NaN: the first tile's, and far from zero): no running maximum, exp or
  // rescale of O in the others.  Pair x of the tile's weights, `less` from their exponents: rounded to 16
  // bits for the matrix product; the sum takes the rounded weights, so that they still average to one.
  template <int NB>
  __device__ __forceinline__ void weight_pair(const f32x16 (&s)[NB], int x, uint32_t (&p)[8 * NB], float (&sum)[2], float less) const {
    const float w0 = fast_exp2(__builtin_fmaf(s[x >> 3][2 * (x & 7)], c0, -less));
    const float w1 = fast_exp2(__builtin_fmaf(s[x >> 3][2 * (x & 7) + 1], c0, -less));
    p[x] = E::pack(w0, w1);
    sum[x & 1] = E::sum2(p[x], sum[x & 1]);
  }

  // The tile's sum of weights accepted, or the reference point moved and the weights formed again.
  template <int NB>
  __device__ __forceinline__ void settle(f32x16 (&s)[NB], uint32_t (&p)[8 * NB], float (&sum)[2]) {
    if (__builtin_expect(__any(!(sum[0] + sum[1] <= limit)), 0)) {
      float mx = s[0][0];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int x = 0; x < 16; ++x) mx = fmaxf(mx, s[kb][x]);
      mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
      float w[1];
      rescale({m}, mx, c0, shift, w);
      m = mx;
      mc = reference(m, c0, shift);
      l *= w[0];
#pragma unroll
      for (int db = 0; db < T::DB; ++db)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[db][x] *= w[0];
      const bool far = mc != mc;
      if (__any(far)) {
        const float from = far ? m : 0.f;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int x = 0; x < 16; ++x) s[kb][x] -= from;
      }
      sum[0] = sum[1] = 0.f;
#pragma unroll
      for (int x = 0; x < 8 * NB; ++x) weight_pair<NB>(s, x, p, sum, far ? shift : mc);
    }
    l += sum[0] + sum[1];
  }

  // V^T operand x = c2 DB + db of a tile: keys 16 c2 + 8 (e / 4) + 4 half + e % 4 (the order of P^T), dim
  // 32 db + li.  A 16-lane group of the transposing read takes 4 keys x 16 dims.
  static __device__ __forceinline__ u32x4 value_operand(const uint8_t* vt, int x) {
    const int lane = threadIdx.x & 63, grp = lane >> 4, ekey = (lane & 15) >> 2, q4 = lane & 3;
    const int c2 = x / T::DB, d = 32 * (x % T::DB) + 16 * (grp & 1) + 4 * q4;
    u32x2 part[2];
#pragma unroll
    for (int rd = 0; rd < 2; ++rd) {
      const int key = 16 * c2 + 8 * rd + 4 * (grp >> 1) + ekey;
      const uint8_t* at = vt + key * T::kRow + (T::vpiece(key, d >> 3) << 4) + ((d >> 2) & 1) * 8;
      part[rd] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16p*)at));
    }
    return u32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
  }

  // O^T += V^T P^T, the operands read kAhead products before they are taken.  `between(x)` is issued
  // after product x.
  template <int NB, class F>
  __device__ __forceinline__ void gather(const uint32_t (&p)[8 * NB], const uint8_t* vt, F between) {
    constexpr int kAll = 2 * NB * T::DB, kAhead = kAll < 4 ? kAll : 4;
    u32x4 v[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) v[x] = value_operand(vt, x);
#pragma unroll
    for (int x = 0; x < kAll; ++x) {
      const int c2 = x / T::DB, db = x % T::DB;
      o[db] = E::mfma(v[x % kAhead], u32x4{p[4 * c2], p[4 * c2 + 1], p[4 * c2 + 2], p[4 * c2 + 3]}, o[db]);
      if (x + kAhead < kAll) v[x % kAhead] = value_operand(vt, x + kAhead);
      between(x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // A tile's weights in one go.
  template <int NB>
  __device__ __forceinline__ void weights(f32x16 (&s)[NB], uint32_t (&p)[8 * NB]) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 8 * NB; ++x) weight_pair<NB>(s, x, p, sum, mc);
    settle<NB>(s, p, sum);
  }

  // A weight of zero does not keep a NaN or an infinity out of a sum, so the tiles that only some of the rows see leave in a
  // row's sums what keys hidden from it hold.  They come first; after them, the sums that are not finite are formed again, from
  // the visible values alone: by the wave, row by row, keys top KT .. +KT - 1, (top - step) KT .., down to `end` KT, a lane each
  // for the products, lanes over the dims for the sums.
  template <int KT, class A>
  __device__ __forceinline__ void without_hidden(const A& a, const PackedPlan& pl, const Seq& s, int r0, int hk,
                                                 int top, int end, int step) {
    float probe[4] = {0.f, 0.f, 0.f, 0.f};                   // zero where all are finite, NaN otherwise
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) probe[x & 3] = __builtin_fmaf(o[db][x], 0.f, probe[x & 3]);
    const float f = (probe[0] + probe[1]) + (probe[2] + probe[3]);
    const int lane = threadIdx.x & 63, half = lane >> 5, li = lane & 31;
    const uint64_t not_finite = __ballot(!(f == 0.f) && r0 + li < s.lq * pl.G);
    const KeyRows<A> key(a, s, hk);
#pragma unroll 1
    for (uint32_t rows = (uint32_t)not_finite | (uint32_t)(not_finite >> 32); rows != 0; rows &= rows - 1) {
      const int own = __builtin_ctz(rows), last = last_key(s, a.causal, r0 + own, pl);
      const uint16_t* qr = (const uint16_t*)a.q + row_at(s, pl, hk, r0 + own, a.q_s);
      const float far = __shfl(mc, own), from = far != far ? __shfl(m, own) : 0.f, less = far != far ? shift : far;
      float sum[2] = {0.f, 0.f};
#pragma unroll 1
      for (int t = top; t >= end; t -= step) {
        const int n = min(KT, last + 1 - t * KT);            // visible keys of the tile
        if (n <= 0) continue;
        const uint16_t* kr = key.k(t * KT + min(lane, n - 1));
        float x = 0.f;
#pragma unroll 1
        for (int d = 0; d < a.D; d += 8) {
          const u32x4 qd = ld16(qr + d), kd = ld16(kr + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x += E::to_float((uint16_t)qd[e]) * E::to_float((uint16_t)kd[e]);
            x += E::to_float((uint16_t)(qd[e] >> 16)) * E::to_float((uint16_t)(kd[e] >> 16));
          }
        }
        x = pl.c0 < 0.f ? -x : x;
        const float w = E::to_float(E::from_float(fast_exp2(__builtin_fmaf(x - from, c0, -less))));
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          const float wj = __shfl(w, j);
          const uint16_t* vr = key.v(t * KT + j);
          if (lane < a.D) sum[0] += wj * E::to_float(vr[lane]);
          if (lane + 64 < a.D) sum[1] += wj * E::to_float(vr[lane + 64]);
        }
      }
#pragma unroll
      for (int db = 0; db < T::DB; ++db)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int d = 32 * db + 8 * (x >> 2) + 4 * half + (x & 3);
          const float y = __shfl(sum[db >> 1], d & 63);
          o[db][x] = li == own ? y : o[db][x];
          if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);                 // (few registers)
        }
    }
  }
};

// One K or V tile of a sequence on its way from global memory to LDS through registers: NT threads,
// KT keys.  Rows past the sequence and dims past D arrive as zeros.
template <class A, int KC, int KT, int NT>
struct Stage;

// What the tiles of K and V have in common, of the tile that is loaded next: of rows of one tensor nothing.
template <class A, int KT, int NT>
struct Pages {
  __device__ __forceinline__ Pages(const A&, const Seq&, int) {}
  __device__ __forceinline__ void fetch(int) {}
};

template <int KC, int KT, int NT>
struct Stage<sf_packed_attention_args, KC, KT, NT> {
  using T = Dims<KC>;
  static constexpr int kPiecesAll = KT * T::kPieces;
  static constexpr int kN = (kPiecesAll + NT - 1) / NT;
  // a thread's pieces lie whole rows apart: one offset, and kStep rows from piece to piece
  static constexpr bool kSteps = NT % T::kPieces == 0;
  static constexpr int kStep = NT / T::kPieces;
  uint32_t off[kSteps ? 1 : kN];                             // global byte offsets in the tile
  const char* base;
  int64_t row;                                               // bytes between rows
  int dbytes;
  u32x4 data[kN];

  __device__ __forceinline__ void init(const sf_packed_attention_args& a, const void* p, const int64_t (&stride)[2], const Seq& s, int hk, int t) {
    base = (const char*)((const uint16_t*)p + (int64_t)s.k0 * stride[0] + (int64_t)hk * stride[1]);
    row = stride[0] * 2;
    dbytes = a.D * 2;
    const int D = a.D;
#pragma unroll
    for (int u = 0; u < (kSteps ? 1 : kN); ++u) {
      const int idx = u * NT + t, key = idx / T::kPieces, piece = idx % T::kPieces;
      off[u] = idx < kPiecesAll && piece * 8 < D ? (uint32_t)(key * row) + piece * 16 : kOutside;
    }
  }
  // tile starting at key j0, keys j0 .. lk - 1 exist (j0 < lk); zeros, and nothing read, where the tile
  // is not `there`: no branch around the loads, so that their registers have one value on every path
  template <class P>
  __device__ __forceinline__ void load(const P&, int j0, int lk, bool there) {
    const int n = min(KT, lk - j0);
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(base + j0 * row, there ? (n - 1) * row + dbytes : 0);
    uint32_t step = (uint32_t)(kStep * row);
    asm volatile("" : "+s"(step));                           // (formed per tile: kept over the loop, the sums cost registers)
#pragma unroll
    for (int u = 0; u < kN; ++u)
      data[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(kSteps ? off[0] + u * step : off[u]), 0, 0));
  }
  template <bool V>
  __device__ __forceinline__ void store(uint8_t* lds, int t) const {
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      const int idx = u * NT + t, key = idx / T::kPieces, piece = idx % T::kPieces;
      if (kPiecesAll % NT == 0 || idx < kPiecesAll)
        st16(lds + key * T::kRow + ((V ? T::vpiece(key, piece) : T::kpiece(key, piece)) << 4), data[u]);
    }
  }
};

// The pages of the units that a wave loads of a tile: UN units of RU consecutive rows.
template <int KT, int NT>
struct Pages<PagedArgs, KT, NT> {
  static constexpr int kWaves = NT / 64, RU = kWaves > KT / 16 ? KT / kWaves : 16, UN = KT / RU / kWaves;
  static_assert(UN >= 1 && RU * UN * kWaves == KT && (RU == 8 || RU == 16), "whole units of 8 or 16 rows");
  typedef __attribute__((address_space(4))) const int32_t constant_i32;
  const int32_t* table;
  PageDiv div;
  int cols, units, first;                                    // units of 16 rows a page; the wave's first row of a tile
  int id[UN], row[UN];                                       // of the next tile: page, first row in it

  __device__ __forceinline__ Pages(const PagedArgs& a, const Seq& s, int wave)
      : table(a.table + s.k0 * a.table_s), div(a.div), cols(a.table_cols), units(a.page_rows >> 4), first(wave * UN * RU) {}
  __device__ __forceinline__ void fetch(int j0) {
#pragma unroll
    for (int x = 0; x < UN; ++x) {
      const int j = max(j0, 0) + first + x * RU, unit = j >> 4, page = page_of(div, unit);
      id[x] = *(constant_i32*)(uintptr_t)(table + min(page, cols - 1));
      row[x] = ((unit - page * units) << 4) + (j & 15);
    }
  }
};

// A tile of a paged cache: each wave loads whole units, so that a unit's page is one scalar base, whatever lies beside it.
template <int KC, int KT, int NT>
struct Stage<PagedArgs, KC, KT, NT> {
  using T = Dims<KC>;
  using P = Pages<PagedArgs, KT, NT>;
  static constexpr int UN = P::UN, RU = P::RU, kUnit = RU * T::kPieces, LU = (kUnit + 63) / 64, kN = UN * LU;
  static constexpr bool kSteps = 64 % T::kPieces == 0;
  static constexpr int kStep = 64 / T::kPieces;
  uint32_t off[kSteps ? 1 : LU];                             // global byte offsets in the unit
  const char* base;
  int64_t page;                                              // bytes between pages, rows
  uint32_t line;
  int dbytes, pages, first;
  u32x4 data[kN];

  __device__ __forceinline__ void init(const PagedArgs& a, const void* p, const int64_t (&stride)[3], const Seq&, int hk, int t) {
    base = (const char*)((const uint16_t*)p + hk * stride[2]);
    page = stride[0] * 2;
    line = (uint32_t)stride[1] * 2;
    dbytes = a.D * 2;
    pages = (int)a.pages;
    first = __builtin_amdgcn_readfirstlane(t >> 6) * UN * RU;
#pragma unroll
    for (int u = 0; u < (kSteps ? 1 : LU); ++u) {
      const int idx = u * 64 + (t & 63), key = idx / T::kPieces, piece = idx % T::kPieces;
      off[u] = idx < kUnit && piece * 8 < a.D ? key * line + piece * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void load(const P& p, int j0, int lk, bool there) {
    uint32_t step = kStep * line;
    asm volatile("" : "+s"(step));
#pragma unroll
    for (int x = 0; x < UN; ++x) {
      const int n = min(RU, lk - (j0 + first + x * RU));
      const bool some = there && n > 0 && (uint32_t)p.id[x] < (uint32_t)pages;
      const __amdgpu_buffer_rsrc_t r = rows_rsrc(base + (some ? p.id[x] * page + (uint64_t)(uint32_t)p.row[x] * line : 0),
                                                 some ? (n - 1) * (int64_t)line + dbytes : 0);
#pragma unroll
      for (int u = 0; u < LU; ++u)
        data[x * LU + u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(kSteps ? off[0] + u * step : off[u]), 0, 0));
    }
  }
  template <bool V>
  __device__ __forceinline__ void store(uint8_t* lds, int t) const {
#pragma unroll
    for (int x = 0; x < UN; ++x)
#pragma unroll
      for (int u = 0; u < LU; ++u) {
        const int idx = u * 64 + (t & 63), key = first + x * RU + idx / T::kPieces, piece = idx % T::kPieces;
        if (kUnit % 64 == 0 || idx < kUnit)
          st16(lds + key * T::kRow + ((V ? T::vpiece(key, piece) : T::kpiece(key, piece)) << 4), data[x * LU + u]);
      }
  }
};

// Keys of a tile straight into the registers of the matrix operand (packed_stream_kernel): keys 32 kb + li, dims
// 16 kk + 8 half .. +7.
template <class A, int KC, int NB>
struct KeyOperand;
template <int KC, int NB>
struct KeyOperand<sf_packed_attention_args, KC, NB> {
  const char* base;
  int64_t row;
  uint32_t off;
  int D, lk;
  u32x4 f[NB][KC];
  __device__ __forceinline__ KeyOperand(const sf_packed_attention_args& a, const Seq& s, int hk) {
    const int half = (threadIdx.x >> 5) & 1, li = threadIdx.x & 31;
    base = (const char*)((const uint16_t*)a.k + (int64_t)s.k0 * a.k_s[0] + (int64_t)hk * a.k_s[1]);
    row = a.k_s[0] * 2;
    off = (uint32_t)(li * row) + 16 * half;
    D = a.D;
    lk = s.lk;
  }
  template <class P>
  __device__ __forceinline__ void load(const P&, int j0, bool there) {
    const int half = (threadIdx.x >> 5) & 1;
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(base + j0 * row, there ? (min(32 * NB, lk - j0) - 1) * row + D * 2 : 0);
    uint32_t o = off, oh = half ? kOutside : off;            // steps that both halves have, that the first has
    asm volatile("" : "+v"(o), "+v"(oh));                    // (formed per tile: kept over the loop, the sums cost registers)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int kk = 0; kk < KC; ++kk)
        f[kb][kk] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            r, (int)((16 * kk + 8 < D ? o : 16 * kk < D ? oh : kOutside) + kb * 32 * (uint32_t)row + 32 * kk), 0, 0));
  }
};
// Of a paged cache: 16 rows have one page, 32 lanes two of them, found a tile ahead with those of V.  Rows past the sequence read
// what their page holds (they are hidden), rows of a page that does not exist zeros.
template <int KC, int NB>
struct KeyOperand<PagedArgs, KC, NB> {
  const char* base;
  int64_t page;
  uint32_t line, off;
  int D, pages;
  u32x4 f[NB][KC];
  // chunks that are whole for every D of this KC
  static constexpr int kWhole = (KC == 2 ? 8 : KC == 3 ? 40 : KC == 4 ? 56 : KC == 6 ? 72 : 104) / 16;
  __device__ __forceinline__ KeyOperand(const PagedArgs& a, const Seq&, int hk)
      : base((const char*)((const uint16_t*)a.k + hk * a.k_s[2])), page(a.k_s[0] * 2), line((uint32_t)a.k_s[1] * 2),
        off((threadIdx.x & 15) * ((uint32_t)a.k_s[1] * 2)), D(a.D), pages((int)a.pages) {}
  __device__ __forceinline__ void load(const Pages<PagedArgs, 32 * NB, 64>& p, int, bool there) {
    const int half = (threadIdx.x >> 5) & 1;
    const bool second = threadIdx.x & 16;
    if (!there) return;                                      // (uniform; what the registers hold is not used)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      uint64_t at[2];
      uint32_t rows[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int id = p.id[2 * kb + x];
        const bool exists = (uint32_t)id < (uint32_t)pages;
        at[x] = (uint64_t)(uintptr_t)(exists ? base + id * page + (uint64_t)(uint32_t)p.row[2 * kb + x] * line : reinterpret_cast<const char*>(kZeros));
        rows[x] = exists ? 0xffffffffu : 0u;
      }
      const char* const q = reinterpret_cast<const char*>((uintptr_t)(second ? at[1] : at[0])) + ((off & (second ? rows[1] : rows[0])) + 16 * half);
#pragma unroll
      for (int kk = 0; kk < KC; ++kk)
        f[kb][kk] = ld16(kk < kWhole || 16 * kk + 8 * half < D ? q + 32 * kk : reinterpret_cast<const char*>(kZeros));
    }
  }
};

// Workgroups of KG groups of NW waves: a wave has 32 rows, the groups have the same rows and take turns at the K/V
// tiles of 64 keys.  A group has two LDS buffers and one barrier a tile; the tile after the next is in flight to
// registers meanwhile.  Tiles go from the last that the rows see to the first, the partly visible ones
// first.  S^T = K Q^T leaves a lane the weights of one row in the very layout that O^T += V^T P^T takes them in,
// so they never pass through LDS; V is turned by its LDS read.
//
// Bound by the issue of matrix products and of the weights' vector instructions, which overlap little: 64 keys x 32 rows
// of 128 dims take 435 and 249 ns, together 577 in a loop of registers alone (64 dims: 218, 237, 406).  A prompt of 16384,
// 32 / 8 heads of 128, causal, bf16: 1.83 to 2.03 ms from card to card, 1.20 to 1.08 PFLOP/s (bf16 products of 8192^3:
// 1.2 to 1.4), of 4096 134 to 143 us; 1.52 ms where all inputs are zero, which draw less power.  8192 tokens, 16
// heads of 64: 168 to 177 us, 0.82 to 0.78 PFLOP/s.
template <class A, class E, int KC, int NW, int KG, bool SHARE = false>
__global__ __launch_bounds__(64 * NW * KG, 2) void packed_tile_kernel(const A a, const PackedPlan pl) {
  using T = Dims<KC>;
  constexpr int kTile = 64 * T::kRow, R = 32 * NW;
  __shared__ __attribute__((aligned(1024))) uint8_t shared[KG * 4 * kTile];          // a group: two buffers of K, V
  const int tid = threadIdx.x % (64 * NW), lane = tid & 63, half = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * NW));
  uint8_t* const smem = shared + group * 4 * kTile;
  // the key heads of one tile are neighbours, so that with 8 of them each XCD keeps to its own K and V
  const int block = workgroup(), hk = block % a.Hkv, rest = block / a.Hkv;
  int slice = rest % pl.slices, slices = pl.slices;
  const int idx = rest / pl.slices;
  Seq s;
  int tile, ntiles;
  bool there;
  // The rows with the most keys first, so that the last workgroups to start are short (8 prompts of 1 to 2048, 16 heads
  // of 64: 42 us, sequence by sequence 47; 10 proteins of 20 to 1024, 16 heads of 48: 24.8 / 26.9).  Of more than
  // 64 sequences there are enough workgroups after any of them.
  if constexpr (SHARE) {
    int slot;
    there = a.B <= 64 ? find_slice<R, 1>(a, pl, 64 * KG, idx, s, tile, slot, slice, slices)
                      : find_slice<R, 4>(a, pl, 64 * KG, idx, s, tile, slot, slice, slices);
    if (hk + (int)threadIdx.x == 0 && slot < pl.tiles && (!there || slice == 0)) note_tile(pl, slot, there && slices > 1, s, tile, idx, slices);
  } else if (a.B > 1 && a.B <= 64) {                           // (SHARE is a kernel of its own: its code here slowed the other by 5%)
    there = find_longest<R>(a, pl, idx, s, tile);
  } else {
    there = find_tile<R>(a, pl, idx, s, tile, ntiles);
    tile = ntiles - 1 - tile;
  }
  if (!SHARE && pl.slices > 1 && hk + slice + (int)threadIdx.x == 0) note_tile(pl, idx, there, s, tile, idx * pl.slices, pl.slices);
  if (!there) return;
  const int rows = s.lq * pl.G, r0 = tile * R + wave * 32;
  const int row = min(r0 + li, rows - 1);                    // rows past the end repeat the last
  const int seen = last_key(s, a.causal, min(tile * R + R, rows) - 1, pl) + 1;   // keys the workgroup's last row sees
  const int n_all = (seen + 63) / 64;
  const int per = (n_all + slices - 1) / slices, t_lo = min(slice * per, n_all), t_hi = min(t_lo + per, n_all);

  RowState<E, KC> st;
  st.init(a, pl, s, row, hk);
  const int mine = last_key(s, a.causal, row, pl);
  // of this wave's rows: the fewest and the most keys
  const int low = __builtin_amdgcn_readfirstlane(last_key(s, a.causal, min(r0, rows - 1), pl));
  const int high = r0 < rows ? __builtin_amdgcn_readfirstlane(last_key(s, a.causal, min(r0 + 31, rows - 1), pl)) : -1;

  if (t_lo < t_hi) {
    Stage<A, KC, 64, 64 * NW> ks, vs;
    Pages<A, 64, 64 * NW> pages(a, s, wave);                 // of the next tile to load
    ks.init(a, a.k, a.k_s, s, hk, tid);
    vs.init(a, a.v, a.v_s, s, hk, tid);
    // this group's tiles t, t - KG, .. (all groups go as many steps: a last tile below t_lo is not read and has no weight)
    int t = t_hi - 1 - group;
    const int t_end = t_lo - group;
    const auto buffer = [&]() __attribute__((always_inline)) { return (t >> (KG - 1)) & 1; };      // of tile t
    pages.fetch(64 * t);
    ks.load(pages, 64 * t, s.lk, t >= t_lo);
    vs.load(pages, 64 * t, s.lk, t >= t_lo);
    pages.fetch(64 * (t - KG));
    const auto kt = [&](int buf) __attribute__((always_inline)) { return smem + buf * 2 * kTile; };
    const auto vt = [&](int buf) __attribute__((always_inline)) { return smem + buf * 2 * kTile + kTile; };
    ks.template store<false>(kt(buffer()), tid);
    vs.template store<true>(vt(buffer()), tid);
    ks.load(pages, 64 * (t - KG), s.lk, t - KG >= t_lo);
    vs.load(pages, 64 * (t - KG), s.lk, t - KG >= t_lo);
    pages.fetch(64 * (t - 2 * KG));
    lds_only_barrier();
    for (; t >= t_end && 64 * t > high; t -= KG) {           // tiles that none of this wave's rows sees
      ks.template store<false>(kt(buffer() ^ 1), tid);
      vs.template store<true>(vt(buffer() ^ 1), tid);
      ks.load(pages, 64 * (t - 2 * KG), s.lk, t - 2 * KG >= t_lo);
      vs.load(pages, 64 * (t - 2 * KG), s.lk, t - 2 * KG >= t_lo);
      pages.fetch(64 * (t - 3 * KG));
      lds_only_barrier();
    }
    const int top = t;
    int hidden = a.causal ? max(t_lo, (low + 1) >> 6) + KG - 1 : -KG;        // once there, the group's tiles left are seen to their end
    // (the buffers as constants: LDS addresses are formed once)
    auto step = [&](auto constant) __attribute__((always_inline)) {
      constexpr int B = decltype(constant)::value;
      f32x16 sc[2];
      // meanwhile the next tile goes to the other buffer, and the one after it is asked for
      st.template products<2>(kt(B), sc, [&](int x) __attribute__((always_inline)) {
        if (x == 0) ks.template store<false>(kt(B ^ 1), tid);
        if (x == 1) vs.template store<true>(vt(B ^ 1), tid);
        if (x == 2) ks.load(pages, 64 * (t - 2 * KG), s.lk, t - 2 * KG >= t_lo);
        if (x == 3) vs.load(pages, 64 * (t - 2 * KG), s.lk, t - 2 * KG >= t_lo);
        if (x == 3) pages.fetch(64 * (t - 3 * KG));
      });
      if (64 * t + 63 > low || (KG > 1 && t < t_lo)) st.template hide<2>(sc, KG > 1 && t < t_lo ? -1 : mine - 64 * t);
      uint32_t p[16];
      st.template weights<2>(sc, p);
      st.template gather<2>(p, vt(B), [](int) {});
      if (__builtin_expect(t <= hidden, 0)) {
        st.template without_hidden<64>(a, pl, s, r0, hk, top, max(t, t_lo), KG);
        hidden = -KG;
      }
      lds_only_barrier();
      t -= KG;
    };
    if (t >= t_end && buffer() != 0) step(std::integral_constant<int, 1>{});
    while (t >= t_end) {
      step(std::integral_constant<int, 0>{});
      if (t < t_end) break;
      step(std::integral_constant<int, 1>{});
    }
    if constexpr (KG > 1) {
      // the second group's sums, lane by lane, to the first
      f32x4* const so = reinterpret_cast<f32x4*>(shared) + wave * 64 * (4 * T::DB + 1) + lane;
      if (group == 1) {
#pragma unroll
        for (int x = 0; x < 4 * T::DB; ++x)
          so[64 * x] = f32x4{st.o[x / 4][4 * (x % 4)], st.o[x / 4][4 * (x % 4) + 1], st.o[x / 4][4 * (x % 4) + 2], st.o[x / 4][4 * (x % 4) + 3]};
        so[64 * 4 * T::DB] = f32x4{st.m, st.l, 0.f, 0.f};
      }
      lds_only_barrier();
      if (group == 0) {
        const f32x4 ml = so[64 * 4 * T::DB];
        const float m = fmaxf(st.m, ml[0]);
        float w[2];
        rescale({st.m, ml[0]}, m, st.c0, st.shift, w);
        st.m = m;
        st.l = st.l * w[0] + ml[1] * w[1];
#pragma unroll
        for (int x = 0; x < 4 * T::DB; ++x) {
          const f32x4 o = so[64 * x];
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[x / 4][4 * (x % 4) + e] = st.o[x / 4][4 * (x % 4) + e] * w[0] + o[e] * w[1];
        }
      }
    }
  }
  if (r0 >= rows || group > 0) return;                       // (no barrier from here on)
  const float l = st.l + __shfl_xor(st.l, 32);
  if (slices > 1) {
    float* po = pl.part + (int64_t)block * R * (T::DP + 2);
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4)
        *reinterpret_cast<f32x4*>(po + (wave * 32 + li) * T::DP + 32 * db + 8 * c4 + 4 * half) =
            f32x4{st.o[db][4 * c4], st.o[db][4 * c4 + 1], st.o[db][4 * c4 + 2], st.o[db][4 * c4 + 3]};
    if (half == 0) *reinterpret_cast<f32x2*>(po + R * T::DP + 2 * (wave * 32 + li)) = f32x2{st.m, l};
    return;
  }
  const float inv = mine < 0 ? 0.f : 1.f / l;
  uint16_t* op = (uint16_t*)a.out + row_at(s, pl, hk, row, a.o_s);
  const bool write = r0 + li < rows;
#pragma unroll
  for (int db = 0; db < T::DB; ++db)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t w[4];                                         // dims 32 db + 16 c + {0, 8} + 4 half .. +3
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = E::pack(st.o[db][8 * c + 2 * e] * inv, st.o[db][8 * c + 2 * e + 1] * inv);
      // half 0 takes the 8 dims 16 c .., half 1 the 8 dims 16 c + 8 ..
      const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      const int d0 = 32 * db + 16 * c + 8 * half;
      if (write && d0 < a.D) st16(op + d0, u32x4{x[0], y[0], x[1], y[1]});
    }
}

// 32 rows a workgroup (a new token's heads, short pieces): its 4 waves each stream a slice of the
// keys, no barrier until the slices are joined: K straight into the registers of the matrix operand,
// V through registers to LDS of the wave's own.  With few rows the keys are split over workgroups too, joined by
// packed_combine_kernel.  Bound by the reads of K and V: 64 tokens over caches of 2048, 32 / 8 heads of 128, 537 MB in 114
// us, 4.7 TB/s; where there is less, by start, join and the latency of their loads: one token over 65536 keys, 16 / 2 heads, 67
// MB in 21.7 us, of which the join is 5.
template <class A, class E, int KC>
__global__ __launch_bounds__(256, 2) void packed_stream_kernel(const A a, const PackedPlan pl) {
  using T = Dims<KC>;
  constexpr int KT = T::DP <= 64 ? 64 : 32, NB = KT / 32, kTile = KT * T::kRow;
  constexpr int kWave = kTile > 32 * T::DP * 4 ? kTile : 32 * T::DP * 4;   // V tile, later the wave's O
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kWave];
  __shared__ f32x2 ml[4][32];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = workgroup(), hk = block % a.Hkv, item = block / a.Hkv;
  Seq s;
  int tile, slice, slices;
  if (pl.share > 0) {
    int slot;
    const bool there = a.B <= 64 ? find_slice<32, 1>(a, pl, 4 * KT, item, s, tile, slot, slice, slices)
                                 : find_slice<32, 4>(a, pl, 4 * KT, item, s, tile, slot, slice, slices);
    if (hk + tid == 0 && slot < pl.tiles && (!there || slice == 0)) note_tile(pl, slot, there && slices > 1, s, tile, item, slices);
    if (!there) return;
  } else {
    int ntiles;
    slice = 0;
    slices = 1;
    if (!find_tile<32>(a, pl, item, s, tile, ntiles)) return;
  }
  const int rows = s.lq * pl.G, r0 = tile * 32;
  const int row = min(r0 + li, rows - 1);
  const int seen = last_key(s, a.causal, min(r0 + 32, rows) - 1, pl) + 1;
  const int n_all = (seen + KT - 1) / KT, Z = slices * 4;
  const int per = (n_all + Z - 1) / Z, t_lo = min((slice * 4 + wave) * per, n_all), t_hi = min(t_lo + per, n_all);
  const int mine = last_key(s, a.causal, row, pl);
  const int low = __builtin_amdgcn_readfirstlane(last_key(s, a.causal, r0, pl));
  uint8_t* vt = smem + wave * kWave;
  {
    RowState<E, KC> st;
    st.init(a, pl, s, row, hk);
    if (t_lo < t_hi) {
      KeyOperand<A, KC, NB> kf(a, s, hk);
      Stage<A, KC, KT, 64> vs;
      Pages<A, KT, 64> pages(a, s, 0);
      vs.init(a, a.v, a.v_s, s, hk, lane);
      pages.fetch(KT * (t_hi - 1));
      kf.load(pages, KT * (t_hi - 1), true);
      vs.load(pages, KT * (t_hi - 1), s.lk, true);
      pages.fetch(KT * (t_hi - 2));
      const int hidden = a.causal ? max(t_lo, (low + 1) / KT) : -1;          // last of the tiles that some rows do not see to their end
      for (int t = t_hi - 1; t >= t_lo; --t) {
        f32x16 sc[NB];
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
          for (int x = 0; x < 16; ++x) sc[kb][x] = 0.f;
#pragma unroll
          for (int kk = 0; kk < KC; ++kk) sc[kb] = E::mfma(kf.f[kb][kk], st.q[kk], sc[kb]);
        }
        vs.template store<true>(vt, lane);
        kf.load(pages, KT * (t - 1), t > t_lo);
        vs.load(pages, KT * (t - 1), s.lk, t > t_lo);
        pages.fetch(KT * (t - 2));
        if (KT * t + KT - 1 > low) st.template hide<NB>(sc, mine - KT * t);
        uint32_t p[8 * NB];
        st.template weights<NB>(sc, p);
        st.template gather<NB>(p, vt, [](int) {});
        if (__builtin_expect(t == hidden, 0)) st.template without_hidden<KT>(a, pl, s, r0, hk, t_hi - 1, t, 1);
      }
    }
    // the slice's O over the wave's tiles, for all threads
    const float l = st.l + __shfl_xor(st.l, 32);
    float* po = (float*)vt;
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4)
        *reinterpret_cast<f32x4*>(po + li * T::DP + 32 * db + 8 * c4 + 4 * half) =
            f32x4{st.o[db][4 * c4], st.o[db][4 * c4 + 1], st.o[db][4 * c4 + 2], st.o[db][4 * c4 + 3]};
    if (half == 0) ml[wave][li] = f32x2{st.m, l};
  }
  lds_only_barrier();
  // thread (row tid / 8, dims 4 (tid % 8) + 32 db): the 4 slices of the waves
  const int jr = tid >> 3, jd = 4 * (tid & 7);
  float m = ml[0][jr][0];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[w][jr][0]);
  float l = 0.f, wt[4];
  rescale({ml[0][jr][0], ml[1][jr][0], ml[2][jr][0], ml[3][jr][0]}, m, fabsf(pl.c0), E::shift(s.lk), wt);
#pragma unroll
  for (int w = 0; w < 4; ++w) l += wt[w] * ml[w][jr][1];
  f32x4 o[T::DB];
#pragma unroll
  for (int db = 0; db < T::DB; ++db) {
    o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>((const float*)(smem + w * kWave) + jr * T::DP + 32 * db + jd);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[db][e] += wt[w] * x[e];
    }
  }
  if (slices > 1) {
    float* po = pl.part + (int64_t)block * 32 * (T::DP + 2);
    if (r0 + jr < rows) {
#pragma unroll
      for (int db = 0; db < T::DB; ++db) *reinterpret_cast<f32x4*>(po + jr * T::DP + 32 * db + jd) = o[db];
      if (jd == 0) *reinterpret_cast<f32x2*>(po + 32 * T::DP + 2 * jr) = f32x2{m, l};
    }
    return;
  }
  const int r = r0 + jr;
  if (r < rows) {
    const float inv = last_key(s, a.causal, r, pl) < 0 ? 0.f : 1.f / l;
    uint16_t* op = (uint16_t*)a.out + row_at(s, pl, hk, r, a.o_s);
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
      if (32 * db + jd < a.D)
        *reinterpret_cast<u32x2*>(op + 32 * db + jd) = u32x2{E::pack(o[db][0] * inv, o[db][1] * inv), E::pack(o[db][2] * inv, o[db][3] * inv)};
  }
}

// Joins the key slices: o = sum_z w_z O_z / sum_z w_z l_z with w_z the worth of slice z's reference point
// against the largest.  LR lanes of 4 dims take a row.  R: rows of a tile; pl.pieces blocks share a
// tile.  From packed_stream_kernel (R = 32: few rows, up to 64 slices) a block takes a row at a time, its
// lane groups the slices z, z + GROUPS, .., joined through LDS; from packed_tile_kernel (few slices) a
// group takes a row and a block 32 of them.  Latency: 4 to 6 us with its launch, whatever it joins up to some MB.
template <class A, class E, int DP, int R>
__global__ __launch_bounds__(256) void packed_combine_kernel(const A a, const PackedPlan pl) {
  constexpr int LR = DP <= 32 ? 8 : DP <= 64 ? 16 : 32, GROUPS = 256 / LR;
  constexpr bool kOneRow = R == 32;
  constexpr int ROWS = kOneRow ? 1 : 32, PASSES = kOneRow ? 1 : ROWS / GROUPS, kBatch = 4;
  const int64_t kStep = (int64_t)a.Hkv * R * (DP + 2);      // from slice to slice
  __shared__ f32x4 so[kOneRow ? GROUPS : 1][LR];
  __shared__ f32x2 sml[GROUPS];
  const int tid = threadIdx.x, lane = tid & 63, group = tid / LR, d = 4 * (tid % LR);
  const int piece = blockIdx.x % pl.pieces, rest = blockIdx.x / pl.pieces, hk = rest % a.Hkv, idx = rest / a.Hkv;
  const int4 f0 = pl.found[2 * idx], f1 = pl.found[2 * idx + 1];
  const Seq s = {f0.x, f0.y, f1.x, f0.z};
  const int slices = f1.z;
  const int rows = s.lq * pl.G, r0 = f0.w * R;
  const float* part = pl.part + ((int64_t)f1.y * a.Hkv + hk) * R * (DP + 2);
  const float c0 = fabsf(pl.c0), shift = E::shift(s.lk);
  for (int in0 = piece * ROWS; in0 < R && r0 + in0 < rows; in0 += pl.pieces * ROWS) {      // (uniform over the block)
    f32x4 o[PASSES];
    float sum[PASSES];
#pragma unroll
    for (int x = 0; x < PASSES; ++x) {
      const int in = kOneRow ? in0 : in0 + x * GROUPS + group;
      const int z0 = kOneRow ? group : 0, dz = kOneRow ? GROUPS : 1;
      const float* ml = part + R * DP + 2 * in;
      const float* po = part + in * DP + d;
      float m = -FLT_MAX, l = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      if (r0 + in < rows && d < DP) {
        for (int z = z0; z < slices; z += kBatch * dz) {
          f32x2 v[kBatch];
          f32x4 ov[kBatch];
#pragma unroll
          for (int y = 0; y < kBatch; ++y) {
            const int64_t at = (z + y * dz < slices ? z + y * dz : z) * kStep;
            v[y] = *reinterpret_cast<const f32x2*>(ml + at);
            ov[y] = *reinterpret_cast<const f32x4*>(po + at);
          }
          // (no use before the last of the loads: left to itself the compiler waited for each in turn, 7.9 us for 4.9)
#pragma unroll
          for (int y = 0; y < kBatch; ++y) asm volatile("" : "+v"(v[y]), "+v"(ov[y]) : : "memory");
          float mz[kBatch + 1], w[kBatch + 1], mx = m;
#pragma unroll
          for (int y = 0; y < kBatch; ++y) {
            if (z + y * dz >= slices) {
              v[y] = f32x2{-FLT_MAX, 0.f};
              ov[y] = f32x4{0.f, 0.f, 0.f, 0.f};             // (whatever it weighs: it may not be finite)
            }
            mz[y] = v[y][0];
            mx = fmaxf(mx, v[y][0]);
          }
          mz[kBatch] = m;
          rescale(mz, mx, c0, shift, w);
          m = mx;
          l *= w[kBatch];
          acc *= w[kBatch];
#pragma unroll
          for (int y = 0; y < kBatch; ++y) {
            l += w[y] * v[y][1];
            acc += w[y] * ov[y];
          }
        }
      }
      if (kOneRow) {                                         // the groups' shares of the row
        so[group][tid % LR] = acc;
        if (d == 0) sml[group] = f32x2{m, l};
        __syncthreads();
        float mg[GROUPS], w[GROUPS];
        m = -FLT_MAX;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          mg[g] = sml[g][0];
          m = fmaxf(m, mg[g]);
        }
        rescale(mg, m, c0, shift, w);
        l = 0.f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          l += w[g] * sml[g][1];
          acc += w[g] * so[g][tid % LR];
        }
        __syncthreads();                                     // (the shares may be overwritten)
      }
      o[x] = acc;
      sum[x] = l;
    }
    if (kOneRow && tid >= 64) continue;
#pragma unroll
    for (int x = 0; x < PASSES; ++x) {
      const int in = kOneRow ? in0 : in0 + x * GROUPS + group, r = r0 + in;
      const bool mine = r < rows && d < a.D && (!kOneRow || tid < LR);
      if (mine) {
        const float inv = last_key(s, a.causal, r, pl) < 0 ? 0.f : 1.f / sum[x];
        *reinterpret_cast<u32x2*>((uint16_t*)a.out + row_at(s, pl, hk, r, a.o_s) + d) =
            u32x2{E::pack(o[x][0] * inv, o[x][1] * inv), E::pack(o[x][2] * inv, o[x][3] * inv)};
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Route {
  int nw;            // waves of rows of packed_tile_kernel's workgroups; 0: packed_stream_kernel
  int groups;        // of such waves, that share the keys
  int kc, dp;
  PackedPlan pl;
  int64_t wgs;
  bool counted;      // packed_starts_kernel counts the tiles
  bool joined() const { return pl.slices > 1 || pl.share > 0; }
};

// What all callers ask of the sizes, queries and types; `what` names the call.
template <class A>
int check_sizes(const A* a, const char* what) {
  if (a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->D <= 0 || a->Tq < 0) {
    sf_set_error("%s: sizes must be positive (B=%d H=%d Hkv=%d D=%d Tq=%lld)", what, a->B, a->H, a->Hkv, a->D, (long long)a->Tq);
    return 1;
  }
  if (a->H % a->Hkv != 0) { sf_set_error("%s: %d heads do not share %d key heads evenly", what, a->H, a->Hkv); return 1; }
  if (a->D > 128 || a->D % 8 != 0) { sf_set_error("%s: head dim %d is not a multiple of 8 up to 128", what, a->D); return 1; }
  if (a->dtype != SF_DTYPE_BF16 && a->dtype != SF_DTYPE_F16) { sf_set_error("%s: element type %d", what, a->dtype); return 1; }
  if (!(fabsf(a->scale) <= 1e30f)) { sf_set_error("%s: scale %g is not finite or above 1e30", what, (double)a->scale); return 1; }
  return 0;
}

// The launch for sequences of about `keys` keys.
template <class A>
int route(const A* a, int64_t keys, Route& r, const char* what) {
  const int G = a->H / a->Hkv;
  r.kc = a->D <= 32 ? 2 : a->D <= 48 ? 3 : a->D <= 64 ? 4 : a->D <= 96 ? 6 : 8;
  r.dp = 32 * ((r.kc + 1) / 2);
  const int64_t rows = a->Tq * G;
  // keys that a row of an average sequence sees, on average
  int64_t seen = keys;
  if (a->causal) seen -= seen < a->Tq / a->B ? seen / 2 : a->Tq / a->B / 2;
  // Up to 64 rows a sequence stream their keys.  Above, tiles of 128 rows; of 256 (half the reads of K and V)
  // where head dims above 64 meet long rows and two workgroups a CU: prompt of 8192, 32 / 8 heads of 128, 128 and 256
  // rows 548 / 512 us, 2048 (256 workgroups) 55 / 75; 8 of 512 41 / 45; 8192, 16 heads of 64 170 / 172.
  r.nw = rows <= 64ll * a->B ? 0 : r.kc > 4 && seen >= 1024 && rows / 256 * a->Hkv >= 512 ? 8 : 4;
  const int R = r.nw ? 32 * r.nw : 32;
  // tiles end at sequence ends: sum_b ceil(rows_b / R) <= rows / R + B
  const int64_t tiles = rows / R + (a->B < rows ? a->B : rows);
  const int64_t full = (rows + R - 1) / R, wgs = (full > a->B ? full : a->B) * a->Hkv;
  int64_t slices = 1, share = 0;
  bool whole = false;
  r.groups = 1;
  if (r.nw) {
    // Few workgroups: two groups of waves share the keys of a workgroup, and workgroups take slices of them, no slice
    // below 512 keys, or 256 on average where the first rows see few (causal without a cache).  Two slices want 1024
    // keys each, for the join.  us with one group and one slice / two groups / groups and slices: prompt of 1024, 16 heads of 64,
    // 18.5 / 15.8 / 20.7 with 2 slices; 2048 31.2 / 24.9; 4096 (512 workgroups) 61 / 52, 4 of 1024 23.3 / 25.3; 2048 of 48,
    // all keys, 29.6 / 25.4 / 38.4; 512 over 8192, 32 / 8 heads of 128, 152 / 119 / 84 with 2, 128 over 8192 144 / 111 / 38 with 8.
    const bool triangle = a->causal && seen * 4 < keys * 3;
    if (r.nw == 4 && (wgs <= 256 ? seen >= 256 : wgs <= 512 && triangle && seen >= 1024)) r.groups = 2;
    slices = 256 / wgs;
    const int64_t most = seen / (triangle ? 256 : 512);
    if (slices > most) slices = most;
    if (slices < 3 && seen < 2048) slices = 1;
    slices = slices < 1 ? 1 : slices > 64 ? 64 : slices;
    // A step that takes tokens of some sequences along with a piece of another: as many slices for each would leave most
    // workgroups with little to do, so they are dealt out by the keys, a workgroup a CU.
    if (kShareTiles<A> && r.nw == 4 && a->B > 1 && a->B <= kShared && !triangle && wgs < 256 && seen >= 1024) {
      r.groups = 2;
      slices = 1;
      share = 256 / a->Hkv;
      if (share < 1) share = 0;
    }
  } else {
    const int64_t least = r.dp > 64 ? 128 : 256;
    // Slices dealt out by the keys, a workgroup a CU or the next multiple of that (one token for 4 caches of 128 to 8192
    // keys, 32 / 8 heads of 128: 16.8 us, as many slices for each 21.6; 32 of them 85 / 126; 100 of 64 to 4096 93 / 141; 384
    // workgroups in place of 256 25 / 20).  From 256 workgroups on only where sequences are uneven and long: of one length
    // the join's launch is lost (4 caches of 4096 20.5 / 20.1, 32 of 4096 108 / 104, 32 of 1024 30 / 28, 256 of 512 129 / 115;
    // 16 of 750 on average, 16 heads of 64, 20.5 / 31.9).
    if (a->B <= kShared && seen >= 2 * least && (wgs < 256 || seen >= 640)) {
      share = 256 * (wgs / 256 + 1) / a->Hkv;
      whole = wgs >= 256;
      // (many key heads of few rows each: the join's buffer, of 32 rows a slice, would exceed 256 MiB)
      if (whole && (share + tiles) * a->Hkv * 32 * (r.dp + 2) > 64 << 20) share = 0;
    }
  }
  r.counted = a->B > kScanned && share == 0;
  // rows of a tile join in blocks of 32, or -- packed_stream_kernel -- one by one, as many blocks as a
  // sequence has rows on average, but few where there are many tiles, most of which need no join
  int64_t pieces = r.nw ? r.nw : (rows + a->B - 1) / a->B;
  if (pieces > 32) pieces = 32;
  if (r.nw == 0) pieces = std::max<int64_t>(std::min(pieces, 1024 / (tiles * a->Hkv)), 1);
  float c0 = a->scale * SF_LOG2E;
  if (fabsf(c0) < FLT_MIN) c0 = FLT_MIN;                     // all logits equal; a masked one stays -inf
  r.pl = PackedPlan{(int)tiles, (int)slices, (int)share, (int)whole, (int)pieces, c0, G, 1.0 / G, nullptr, nullptr, nullptr};
  r.wgs = (share > 0 ? share + tiles : tiles * slices) * a->Hkv;
  if (r.wgs > INT32_MAX || tiles * a->Hkv * 32 > INT32_MAX) { sf_set_error("%s: problem too large for the grid", what); return 1; }
  return 0;
}

template <class A>
size_t part_bytes(const A* a, const Route& r) {
  const size_t starts = r.counted ? ((size_t)a->B + 1) * sizeof(int) : 0;
  if (!r.joined()) return starts;
  const int R = r.nw ? 32 * r.nw : 32;
  return (size_t)r.wgs * R * (r.dp + 2) * sizeof(float) + (size_t)r.pl.tiles * 2 * sizeof(int4);
}

template <class A, class E, int KC>
int launch(const A* a, const Route& r, hipStream_t st) {
  const dim3 grid = r.wgs <= kGridX ? dim3((unsigned)r.wgs) : dim3(kGridX, (unsigned)((r.wgs + kGridX - 1) / kGridX));
  if (r.pl.starts != nullptr) {
    hipLaunchKernelGGL(packed_starts_kernel<A>, dim3(1), dim3(1024), 0, st, *a, r.pl, r.nw ? 32 * r.nw : 32);
    if (sf_check_launch("packed_starts_kernel")) return 1;
  }
  if (r.nw == 0) {
    hipLaunchKernelGGL((packed_stream_kernel<A, E, KC>), grid, dim3(256), 0, st, *a, r.pl);
  } else if (r.nw == 4 && r.pl.share > 0) {
    if constexpr (kShareTiles<A>) hipLaunchKernelGGL((packed_tile_kernel<A, E, KC, 4, 2, true>), grid, dim3(512), 0, st, *a, r.pl);
  } else if (r.nw == 4) {
    if (r.groups == 2) hipLaunchKernelGGL((packed_tile_kernel<A, E, KC, 4, 2>), grid, dim3(512), 0, st, *a, r.pl);
    else hipLaunchKernelGGL((packed_tile_kernel<A, E, KC, 4, 1>), grid, dim3(256), 0, st, *a, r.pl);
  } else if constexpr (KC > 4) {
    hipLaunchKernelGGL((packed_tile_kernel<A, E, KC, 8, 1>), grid, dim3(512), 0, st, *a, r.pl);
  }
  const int rc = sf_check_launch(r.nw ? "packed_tile_kernel" : "packed_stream_kernel");
  if (rc || !r.joined()) return rc;
  const dim3 gc((unsigned)(r.pl.tiles * a->Hkv * r.pl.pieces));
  constexpr int DP = Dims<KC>::DP;                           // (tiles of 256 rows are never sliced)
  if (r.nw) hipLaunchKernelGGL((packed_combine_kernel<A, E, DP, 128>), gc, dim3(256), 0, st, *a, r.pl);
  else hipLaunchKernelGGL((packed_combine_kernel<A, E, DP, 32>), gc, dim3(256), 0, st, *a, r.pl);
  return sf_check_launch("packed_combine_kernel");
}

template <class A, class E>
int launch_type(const A* a, const Route& r, hipStream_t st) {
  switch (r.kc) {
    case 2: return launch<A, E, 2>(a, r, st);
    case 3: return launch<A, E, 3>(a, r, st);
    case 4: return launch<A, E, 4>(a, r, st);
    case 6: return launch<A, E, 6>(a, r, st);
    default: return launch<A, E, 8>(a, r, st);
  }
}

// The call itself: workspace of part_bytes.
template <class A>
int run(const A* a, Route& r, void* workspace, size_t workspace_bytes, void* stream, const char* what) {
  const size_t need = part_bytes(a, r);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    sf_set_error("%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, need, workspace_bytes);
    return 1;
  }
  r.pl.part = static_cast<float*>(workspace);
  if (r.counted) r.pl.starts = static_cast<int*>(workspace);
  r.pl.found = reinterpret_cast<int4*>(r.pl.part + r.wgs * (r.nw ? 32 * r.nw : 32) * (r.dp + 2));
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a->dtype == SF_DTYPE_BF16 ? launch_type<A, Bf16>(a, r, st) : launch_type<A, Fp16>(a, r, st);
}

}  // namespace
