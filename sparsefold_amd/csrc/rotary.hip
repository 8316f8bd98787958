// Rotary positions of query and key heads, with the per-head norm before them in the same pass.
//
//   x' = x                                                       (norm 0)
//   x' = x rsqrt(mean x^2 + eps) w                               (norm 1: rms)
//   x' = (x - mean x) rsqrt(mean (x - mean x)^2 + eps) w + b     (norm 2: layer)
//   y_a = x'_a c - x'_b s,  y_b = x'_b c + x'_a s,  (c, s) = magnitude (cos, sin)(position f_i)
//
// for the pairs (a, b) = (i, i + R/2) or (2i, 2i + 1) of the first R dims; the others keep x'.
//
// Bound by memory: each element is read and written once.  A wave takes one token and some of its
// heads.  It computes the token's R/2 angles once, a lane each, and keeps cos and sin in LDS; a lane
// then owns V pairs (two pieces of V elements) of a head, so that norm and rotation run in registers
// whichever way the pairs lie, and the loads and stores are 16 bytes wide.  The next heads' loads are on their
// way while these are worked on.  8192 tokens, 32 + 8 heads of 128 in fp16, half of the dims: 32 us, 5.2 TB/s (a large
// copy: 5.2); 16384 tokens in bf16 with a norm: 71 us, 4.7 TB/s; up to some hundred tokens 3.4 to 4 us, the launch.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "sf_common.h"

namespace {

constexpr int kMaxPairs = 128;                               // head dims up to 256
constexpr int kWaves = 4;
// A launch dimension holds less than 2^32 threads: workgroups past kGridX continue in the next row of the grid.
constexpr int kGridX = 1 << 22;

struct RotBf16 {
  typedef uint16_t raw;
  static __device__ __forceinline__ float to_float(raw v) { return bf2f(v); }
  static __device__ __forceinline__ raw from_float(float v) { return f2bf(v); }
};
struct RotF16 {
  typedef uint16_t raw;
  static __device__ __forceinline__ float to_float(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ raw from_float(float v) { return __builtin_bit_cast(raw, (_Float16)v); }
};
struct RotF32 {
  typedef float raw;
  static __device__ __forceinline__ float to_float(raw v) { return v; }
  static __device__ __forceinline__ raw from_float(float v) { return v; }
};

// V consecutive elements, one load or store.
template <class E, int V>
struct Piece {
  typedef typename E::raw vec __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ vec load(const typename E::raw* p) { return *reinterpret_cast<const vec*>(p); }
  static __device__ __forceinline__ void widen(const vec& v, float* f) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = E::to_float(v[e]);
  }
  static __device__ __forceinline__ void store(typename E::raw* p, const float* f) {
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = E::from_float(f[e]);
    *reinterpret_cast<vec*>(p) = v;
  }
};
template <class E>
struct Piece<E, 1> {
  typedef typename E::raw vec;
  static __device__ __forceinline__ vec load(const typename E::raw* p) { return *p; }
  static __device__ __forceinline__ void widen(const vec& v, float* f) { f[0] = E::to_float(v); }
  static __device__ __forceinline__ void store(typename E::raw* p, const float* f) { *p = E::from_float(f[0]); }
};

// cos and sin of position * freq.  The angle is reduced to a quarter turn in 64 bits (a far position
// times a fast frequency has no digits left in 32); on |x| <= pi / 4 the Taylor series to x^9 and
// x^10 are off by less than 3e-9.
__device__ __forceinline__ f32x2 cos_sin(double position, double freq) {
  const double t = position * (freq * 0.63661977236758134308);           // quarter turns
  const double n = rint(t);
  const float x = (float)((t - n) * 1.57079632679489661923);
  const int quadrant = (int)(n - 4.0 * floor(n * 0.25));
  const float y = x * x;
  const float sn = x * (1.f + y * (-1.f / 6.f + y * (1.f / 120.f + y * (-1.f / 5040.f + y * (1.f / 362880.f)))));
  const float cs = 1.f + y * (-0.5f + y * (1.f / 24.f + y * (-1.f / 720.f + y * (1.f / 40320.f + y * (-1.f / 3628800.f)))));
  const float c = quadrant & 1 ? sn : cs, s = quadrant & 1 ? cs : sn;
  return f32x2{quadrant == 1 || quadrant == 2 ? -c : c, quadrant >= 2 ? -s : s};
}

struct RotaryPlan {
  int lph;           // lanes of a head (a power of two)
  int per_wave;      // heads of a wave
  int chunks;        // waves of a token
  int pos64;
};

template <class E, int V, int UPL, int NORM, bool INTERLEAVED>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(const sf_rotary_args a, const RotaryPlan pl) {
  typedef typename E::raw raw;
  __shared__ f32x2 table[kWaves][kMaxPairs];
  __shared__ __attribute__((aligned(16))) float affine[NORM == 2 ? 4 : NORM == 1 ? 2 : 1][2 * kMaxPairs];   // weights of q, k, biases of q, k
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = ((int64_t)blockIdx.y * kGridX + blockIdx.x) * kWaves + wave;
  const int64_t token = task / pl.chunks;
  if (NORM != 0) {                                           // read from memory once for all waves
    for (int d = threadIdx.x; d < a.D; d += 64 * kWaves) {
      affine[0][d] = a.q_weight != nullptr ? a.q_weight[d] : 1.f;
      affine[1][d] = a.k_weight != nullptr ? a.k_weight[d] : 1.f;
      if (NORM == 2) {
        affine[2][d] = a.q_bias != nullptr ? a.q_bias[d] : 0.f;
        affine[3][d] = a.k_bias != nullptr ? a.k_bias[d] : 0.f;
      }
    }
    __syncthreads();
  }
  if (token >= a.T) return;                                  // (no barrier from here on)
  const int first = (int)(task - token * pl.chunks) * pl.per_wave, end = min(first + pl.per_wave, a.H + a.Hk);
  const int half_r = a.R >> 1;

  const double position = pl.pos64 ? (double)((const int64_t*)a.positions)[token] : (double)((const int32_t*)a.positions)[token];
#pragma unroll
  for (int i0 = 0; i0 < kMaxPairs; i0 += 64) {
    const int i = i0 + lane;
    if (i < half_r) {
      const f32x2 v = cos_sin(position, a.freqs[i]);
      table[wave][i] = f32x2{v[0] * a.magnitude, v[1] * a.magnitude};
    }
  }
  asm volatile("" ::: "memory");                             // a wave's LDS accesses are in order

  constexpr bool kInPiece = INTERLEAVED && V > 1;            // a pair's two dims lie in one piece
  // ---- this lane's units: V pairs each, or 2 V dims behind the rotated ones ----
  const int sub = lane & (pl.lph - 1), group = lane / pl.lph, step = 64 / pl.lph;
  const int rotating = half_r / V, units = rotating + (a.D - a.R + 2 * V - 1) / (2 * V);
  int at[UPL][2];                                            // first dims of its two pieces (-1: none)
  f32x2 cs[UPL][V];
#pragma unroll
  for (int x = 0; x < UPL; ++x) {
    const int u = sub + 64 * x;
    at[x][0] = at[x][1] = -1;
    if (u < rotating) {
      // the pieces of neighbouring lanes are neighbours: whole lines an instruction, in either layout
      at[x][0] = kInPiece ? V * u : INTERLEAVED ? 2 * u : V * u;
      at[x][1] = kInPiece ? half_r + V * u : INTERLEAVED ? 2 * u + 1 : half_r + V * u;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int pair = !kInPiece ? V * u + e : e < V / 2 ? at[x][0] / 2 + e : at[x][1] / 2 + e - V / 2;
        cs[x][e] = table[wave][pair];
      }
    } else if (u < units) {
      at[x][0] = a.R + V * (u - rotating);
      if (at[x][0] + V * (units - rotating) < a.D) at[x][1] = at[x][0] + V * (units - rotating);
    }
  }

  const float inv_d = 1.f / (float)a.D;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {                  // query heads, then key heads
    const int h0 = which ? max(first - a.H, 0) : first, h1 = which ? end - a.H : min(end, a.H);
    if (h0 >= h1) continue;
    const raw* src = (const raw*)(which ? a.k : a.q) + token * (which ? a.k_s[0] : a.q_s[0]);
    raw* dst = (raw*)(which ? a.k_out : a.q_out) + token * (which ? a.ko_s[0] : a.qo_s[0]);
    const int64_t src_h = which ? a.k_s[1] : a.q_s[1], dst_h = which ? a.ko_s[1] : a.qo_s[1];
    float w[UPL][2][V], b[UPL][2][V];
    if (NORM != 0) {
#pragma unroll
      for (int x = 0; x < UPL; ++x)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int d = max(at[x][p], 0) + e;
            w[x][p][e] = affine[which][d];
            b[x][p][e] = NORM == 2 ? affine[NORM == 2 ? 2 + which : 0][d] : 0.f;
          }
    }
    // the next heads' loads are on their way while these are worked on
    typename Piece<E, V>::vec next[UPL][2];
    auto fetch = [&](int h) __attribute__((always_inline)) {
      const raw* sp = src + (int64_t)min(h, h1 - 1) * src_h;
#pragma unroll
      for (int x = 0; x < UPL; ++x)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (at[x][p] >= 0) next[x][p] = Piece<E, V>::load(sp + at[x][p]);
    };
    fetch(h0 + group);
#pragma unroll 1
    for (int hb = h0; hb < h1; hb += step) {
      const int h = hb + group;
      const bool ok = h < h1;
      float f[UPL][2][V];
#pragma unroll
      for (int x = 0; x < UPL; ++x)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if (at[x][p] >= 0) {
            Piece<E, V>::widen(next[x][p], f[x][p]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) f[x][p][e] = 0.f;
          }
        }
      if (hb + step < h1) fetch(h + step);
      if (NORM != 0) {
        auto each = [&](auto fn) __attribute__((always_inline)) {
#pragma unroll
          for (int x = 0; x < UPL; ++x)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int e = 0; e < V; ++e) fn(f[x][p][e], at[x][p] >= 0);
        };
        auto head_sum = [&](float v) __attribute__((always_inline)) {
          for (int o = 1; o < pl.lph; o <<= 1) v += __shfl_xor(v, o);
          return v;
        };
        // the mean of squares of f, from which a layer norm's mean is taken first
        auto mean_square = [&]() __attribute__((always_inline)) {
          float t = 0.f;
          if (NORM == 2) {
            each([&](float v, bool) { t += v; });
            const float mean = head_sum(t) * inv_d;
            each([&](float& v, bool there) { v -= there ? mean : 0.f; });
            t = 0.f;
          }
          each([&](float v, bool) { t += v * v; });
          return head_sum(t) * inv_d;
        };
        float square = mean_square() + a.eps;
        const bool outside = !(square >= 0x1p-100f && square <= FLT_MAX);
        if (__any(outside)) {
          // sums that pass fp32, or squares that vanish in it: again from the head over a power of two near its largest value (or eps's
          // root), which the norm takes out.  Infinities stay.
          const raw* sp = src + (int64_t)min(h, h1 - 1) * src_h;
          float top = sqrtf(a.eps);
#pragma unroll
          for (int x = 0; x < UPL; ++x)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (at[x][p] >= 0) Piece<E, V>::widen(Piece<E, V>::load(sp + at[x][p]), f[x][p]);
          each([&](float v, bool there) { top = there ? fmaxf(top, fabsf(v)) : top; });
          for (int o = 1; o < pl.lph; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
          const uint32_t exponent = min(max(__float_as_uint(top) >> 23, 1u), 253u);
          const float scale = outside && top <= FLT_MAX ? __uint_as_float((254u - exponent) << 23) : 1.f;
          each([&](float& v, bool there) { v = there ? v * scale : 0.f; });
          square = mean_square() + a.eps * scale * scale;
          if (a.eps > 0.f) square = fmaxf(square, FLT_MIN);                  // (a head of one value: 0)
        }
        const float rs = rsqrtf(square);
#pragma unroll
        for (int x = 0; x < UPL; ++x)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int e = 0; e < V; ++e) f[x][p][e] = f[x][p][e] * rs * w[x][p][e] + b[x][p][e];
      }
#pragma unroll
      for (int x = 0; x < UPL; ++x) {
        float* z = &f[x][0][0];                              // 2 V values: the pieces one after the other
        if (sub + 64 * x < rotating) {                       // (others stay: a turn by 0 would mix an infinity in)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float& za = INTERLEAVED ? z[2 * e] : z[e];
            float& zb = INTERLEAVED ? z[2 * e + 1] : z[V + e];
            const float va = za, vb = zb;
            za = va * cs[x][e][0] - vb * cs[x][e][1];
            zb = vb * cs[x][e][0] + va * cs[x][e][1];
          }
        }
        raw* dp = dst + (int64_t)h * dst_h;
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (ok && at[x][p] >= 0) Piece<E, V>::store(dp + at[x][p], f[x][p]);
      }
    }
  }
}

template <class E, int V, int UPL>
void launch(const sf_rotary_args* a, const RotaryPlan& pl, dim3 grid, hipStream_t st) {
  auto by_layout = [&](auto norm) {
    constexpr int NORM = decltype(norm)::value;
    if (a->interleaved) hipLaunchKernelGGL((rotary_kernel<E, V, UPL, NORM, true>), grid, dim3(64 * kWaves), 0, st, *a, pl);
    else hipLaunchKernelGGL((rotary_kernel<E, V, UPL, NORM, false>), grid, dim3(64 * kWaves), 0, st, *a, pl);
  };
  if (a->norm == SF_NORM_RMS) by_layout(std::integral_constant<int, 1>{});
  else if (a->norm == SF_NORM_LAYER) by_layout(std::integral_constant<int, 2>{});
  else by_layout(std::integral_constant<int, 0>{});
}

}  // namespace

extern "C" int sf_hip_rotary_fwd(const sf_rotary_args* a, void* stream) {
  if (a == nullptr) { sf_set_error("rotary: null args"); return 1; }
  if (a->T < 0 || a->H <= 0 || a->Hk < 0 || a->H > 1 << 24 || a->Hk > 1 << 24 || a->D <= 0 || a->D > 256) {
    sf_set_error("rotary: sizes T=%lld H=%d Hk=%d D=%d (heads positive, up to 2^24; D <= 256)", (long long)a->T, a->H, a->Hk, a->D); return 1;
  }
  if (a->R < 2 || a->R > a->D || a->R % 2 != 0) { sf_set_error("rotary: rotated dims %d are not even and within 2 .. %d", a->R, a->D); return 1; }
  if (a->dtype != SF_DTYPE_BF16 && a->dtype != SF_DTYPE_F16 && a->dtype != SF_DTYPE_F32) { sf_set_error("rotary: element type %d", a->dtype); return 1; }
  if (a->norm != SF_NORM_NONE && a->norm != SF_NORM_RMS && a->norm != SF_NORM_LAYER) { sf_set_error("rotary: norm %d", a->norm); return 1; }
  if (a->T == 0) return 0;
  if (a->q == nullptr || a->q_out == nullptr || a->positions == nullptr || a->freqs == nullptr ||
      (a->Hk > 0 && (a->k == nullptr || a->k_out == nullptr))) {
    sf_set_error("rotary: q, k, their outputs, positions and freqs must be non-null"); return 1;
  }
  // the widest pieces that sizes, strides and addresses allow
  const int size = a->dtype == SF_DTYPE_F32 ? 4 : 2;
  auto fits = [&](int v) {
    const int bytes = v * size;
    if ((a->R / 2) % v != 0 || a->D % v != 0) return false;
    uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->q_out | (uintptr_t)((a->q_s[0] | a->q_s[1] | a->qo_s[0] | a->qo_s[1]) * size);
    if (a->Hk > 0) bits |= (uintptr_t)a->k | (uintptr_t)a->k_out | (uintptr_t)((a->k_s[0] | a->k_s[1] | a->ko_s[0] | a->ko_s[1]) * size);
    return (bits & (uintptr_t)(bytes - 1)) == 0;
  };
  const int v = size == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int units = (a->R / 2) / v + (a->D - a->R + 2 * v - 1) / (2 * v);
  RotaryPlan pl{};
  pl.lph = 1;
  while (pl.lph < units && pl.lph < 64) pl.lph <<= 1;
  const int heads = a->H + a->Hk, at_once = 64 / pl.lph;
  pl.per_wave = heads;
  pl.chunks = (heads + pl.per_wave - 1) / pl.per_wave;
  // few tokens: their heads spread over waves until the GPU is filled; without a norm, whose waves have
  // more to set up, also where it gets another round (8192 tokens, 32 + 8 heads of 128 in fp16, 1 / 5 waves a
  // token: 36.4 / 33.3 us; with a norm, bf16, 16384 tokens, 1 / 2: 71 / 78)
  while (pl.per_wave > at_once && a->T * pl.chunks < (a->norm == SF_NORM_NONE ? 32768 : 4096)) {
    pl.per_wave = (pl.per_wave / 2 + at_once - 1) / at_once * at_once;
    pl.chunks = (heads + pl.per_wave - 1) / pl.per_wave;
  }
  pl.pos64 = a->positions_64;
  const int64_t blocks = (a->T * pl.chunks + kWaves - 1) / kWaves;
  if (blocks > INT32_MAX) { sf_set_error("rotary: problem too large for the grid"); return 1; }
  const dim3 grid = blocks <= kGridX ? dim3((unsigned)blocks) : dim3(kGridX, (unsigned)((blocks + kGridX - 1) / kGridX));
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto by_width = [&](auto type) {
    using E = decltype(type);
    if constexpr (sizeof(typename E::raw) == 2) {
      if (v == 8) return launch<E, 8, 1>(a, pl, grid, st);
    }
    if (v == 4) return launch<E, 4, 1>(a, pl, grid, st);
    if (units <= 64) return launch<E, 1, 1>(a, pl, grid, st);
    return launch<E, 1, 2>(a, pl, grid, st);
  };
  if (a->dtype == SF_DTYPE_BF16) by_width(RotBf16{});
  else if (a->dtype == SF_DTYPE_F16) by_width(RotF16{});
  else by_width(RotF32{});
  return sf_check_launch("rotary_kernel");
}
