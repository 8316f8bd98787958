// The residual's addition and the root-mean-square norm of rows, in the rows' type or microscaled:
//   h = x + residual (rounded to the type),  y = h rsqrt(mean h^2 + eps) weight.
//
// Squares, their sum, the root and the products are 64-bit: the vector units do those at the rate of 32 bits, and memory
// bounds the kernel either way.  So rows of any finite size have a norm, and the codes of 8 and 4 bits, which jump at
// borders, do not depend on the order of the sum.
#include <type_traits>

#include "mx.h"

namespace {

struct Same {};                                              // y in the rows' type

// A double to the nearest float but with the last bit set where something was cut off: rounded again to fewer bits (two
// fewer at least) it gives what rounding the double at once gives.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  const double back = (double)f;
  uint32_t b = __float_as_uint(f);
  b -= fabs(back) > fabs(d) ? 1u : 0u;
  b |= back != d ? 1u : 0u;
  return __uint_as_float(b);
}

// The float that rounds to E as d does.  (By way of the nearest float, 1 of 2^14 results of fp16 comes out on the wrong side of a
// border.)  For fp16, which has nothing below 2^-25, the 29 bits that a float lacks are taken together in its last one: three
// integer instructions, where to_odd takes four of 64 bits (100000 rows of 64: 35.8 us, to_odd 38.8, rounded twice 31.9; rows of
// 4096, which memory bounds, take the same time).
template <class E>
__device__ __forceinline__ float before(double d) {
  if constexpr (std::is_same<E, RowFp32>::value) {
    return (float)d;
  } else if constexpr (std::is_same<E, RowFp16>::value) {
    constexpr uint32_t kRest = (1u << 29) - 1;
    const uint64_t b = __builtin_bit_cast(uint64_t, d);
    const uint32_t lo = (uint32_t)b, some = (lo & kRest) + kRest;              // (bit 29: not zero)
    return (float)__builtin_bit_cast(double, (b & ~0xffffffffull) | (some & (kRest + 1)) | (lo & ~kRest));
  } else {
    return to_odd(d);
  }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Sum over the TPR threads that share a row.  `parts`: [2][waves], used in turn, so that one barrier a row suffices.
template <int TPR>
__device__ __forceinline__ double row_total(double v, double (*parts)[TPR > 64 ? TPR / 64 : 1], int turn) {
  v = wave_sum64(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) parts[turn][threadIdx.x >> 6] = v;
    lds_only_barrier();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += parts[turn][w];
  }
  return v;
}

// TPR threads hold a row, N pieces of 8 elements each; rows in turns, the next one's loads in flight; the weights stay in
// registers.  Bound by memory: 16384 rows of 4096, bf16 with residual, to 8 bits: 93.7 us, 5.0 TB/s; 8 rows 3.3 us, a launch.
template <class E, class F, int TPR, int N>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void add_rms_norm_kernel(const sf_add_rms_norm_args a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kRows = kThreads / TPR;
  typedef typename E::T T;
  __shared__ double parts[2][TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR, sub = kRows == 1 ? 0 : threadIdx.x / TPR, C = a.C;
  const T* const x = (const T*)a.x;
  const T* const res = (const T*)a.residual;
  float w[N][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = 8 * (n * TPR + t);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[n][e] = 1.f;
    if (a.weight != nullptr && c < C) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[n][e] = a.weight[c + e];
    }
  }
  Raw8<E> xr[N], rr[N];
  const auto load = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = 8 * (n * TPR + t);
      if (r < a.R && c < C) {
        xr[n].load(x + r * a.x_rs + c);
        if (res != nullptr) rr[n].load(res + r * a.r_rs + c);
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t r = (int64_t)blockIdx.x * kRows + sub;
  load(r);
  const double inv_c = 1.0 / C;
  // (with more threads than a wave a row, r is uniform over the workgroup: every thread meets every barrier)
  for (int turn = 0; r < a.R; r += step, turn ^= 1) {
    float h[N][8];
    double sq = 0.0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = 8 * (n * TPR + t);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[n][e] = 0.f;
      if (c < C) {
        xr[n].get(h[n]);
        if (res != nullptr) {
          float q[8];
          rr[n].get(q);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[n][e] = E::round(h[n][e] + q[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += (double)h[n][e] * (double)h[n][e];
    }
    load(r + step);
    if (a.sum != nullptr) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = 8 * (n * TPR + t);
        if (c < C) Raw8<E>::store((T*)a.sum + r * a.h_rs + c, h[n]);
      }
    }
    const double rstd = 1.0 / sqrt(row_total<TPR>(sq, parts, turn) * inv_c + (double)a.eps);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = 8 * (n * TPR + t);
      float y[8];
      if (c < C) {
        if constexpr (std::is_same<F, Same>::value) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = before<E>((double)h[n][e] * rstd * (double)w[n][e]);
          Raw8<E>::store((T*)a.y + r * a.y_rs + c, y);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = to_odd((double)h[n][e] * rstd * (double)w[n][e]);
          uint32_t byte;
          const typename F::Codes codes = mx_encode<F>(y, byte);               // (C % 32 == 0: whole quads of lanes)
          *reinterpret_cast<typename F::Codes*>((uint8_t*)a.codes + r * a.c_rs + (int64_t)c / 8 * F::kBytes) = codes;
          if ((t & 3) == 0) ((uint8_t*)a.scales)[r * a.s_rs + (c >> 5)] = (uint8_t)byte;
        }
      }
    }
  }
}

// Rows of any length and alignment, an element at a time, twice over the row.  Bound by the latency of its dependent steps (us beside the
// kernel above: bf16 with residual, 8 rows of 4095 / 4096 11.6 / 4.0, 16384 291 / 104, 100000 of 99 / 96 98 / 46, 2048 of 16392 / 16384 126 / 51).
template <class E>
__global__ __launch_bounds__(256) void add_rms_norm_any_kernel(const sf_add_rms_norm_args a) {
  typedef typename E::T T;
  __shared__ double parts[2][4];
  const T* const res = (const T*)a.residual;
  for (int64_t r = blockIdx.x, turn = 0; r < a.R; r += gridDim.x, turn ^= 1) {
    const T* const x = (const T*)a.x + r * a.x_rs;
    T* const sum = (T*)a.sum + r * a.h_rs;
    T* const y = (T*)a.y + r * a.y_rs;
    double sq = 0.0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      float h = E::load(x + c);
      if (res != nullptr) h = E::round(h + E::load(res + r * a.r_rs + c));
      if (a.sum != nullptr) E::store(sum + c, h);
      sq += (double)h * (double)h;
    }
    const double rstd = 1.0 / sqrt(row_total<256>(sq, parts, (int)turn) / a.C + (double)a.eps);
    for (int c = threadIdx.x; c < a.C; c += 256) {           // (each thread its own elements again: x may have become h)
      float h;
      if (a.sum != nullptr) {
        h = E::load(sum + c);
      } else {
        h = E::load(x + c);
        if (res != nullptr) h = E::round(h + E::load(res + r * a.r_rs + c));
      }
      E::store(y + c, before<E>((double)h * rstd * (a.weight != nullptr ? (double)a.weight[c] : 1.0)));
    }
  }
}

// Microscaled rows longer than registers hold: 8 elements a lane, the row read twice.
template <class E, class F>
__global__ __launch_bounds__(256) void add_rms_norm_long_kernel(const sf_add_rms_norm_args a) {
  typedef typename E::T T;
  __shared__ double parts[2][4];
  const T* const res = (const T*)a.residual;
  for (int64_t r = blockIdx.x, turn = 0; r < a.R; r += gridDim.x, turn ^= 1) {
    const auto element = [&](int c, bool again, float (&h)[8]) __attribute__((always_inline)) {
      Raw8<E> v;
      if (again && a.sum != nullptr) {
        v.load((const T*)a.sum + r * a.h_rs + c);
        v.get(h);
        return;
      }
      v.load((const T*)a.x + r * a.x_rs + c);
      v.get(h);
      if (res != nullptr) {
        float q[8];
        v.load(res + r * a.r_rs + c);
        v.get(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = E::round(h[e] + q[e]);
      }
    };
    double sq = 0.0;
    for (int c = 8 * threadIdx.x; c < a.C; c += 8 * 256) {
      float h[8];
      element(c, false, h);
      if (a.sum != nullptr) Raw8<E>::store((T*)a.sum + r * a.h_rs + c, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += (double)h[e] * (double)h[e];
    }
    const double rstd = 1.0 / sqrt(row_total<256>(sq, parts, (int)turn) / a.C + (double)a.eps);
    for (int c = 8 * threadIdx.x; c < a.C; c += 8 * 256) {
      float h[8], y[8];
      element(c, true, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = to_odd((double)h[e] * rstd * (a.weight != nullptr ? (double)a.weight[c + e] : 1.0));
      uint32_t byte;
      const typename F::Codes codes = mx_encode<F>(y, byte);
      *reinterpret_cast<typename F::Codes*>((uint8_t*)a.codes + r * a.c_rs + (int64_t)c / 8 * F::kBytes) = codes;
      if ((threadIdx.x & 3) == 0) ((uint8_t*)a.scales)[r * a.s_rs + (c >> 5)] = (uint8_t)byte;
    }
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class E, class F, int TPR, int N>
int launch(const sf_add_rms_norm_args* a, hipStream_t st) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  const int64_t groups = (a->R + kThreads / TPR - 1) / (kThreads / TPR);
  const int resident = sf_resident_workgroups(reinterpret_cast<const void*>(add_rms_norm_kernel<E, F, TPR, N>), kThreads);
  hipLaunchKernelGGL((add_rms_norm_kernel<E, F, TPR, N>), dim3((unsigned)(groups < resident ? groups : resident)), dim3(kThreads), 0, st, *a);
  return sf_check_launch("add_rms_norm_kernel");
}

template <class E, class F>
int launch_rows(const sf_add_rms_norm_args* a, hipStream_t st) {
  const int pieces = (a->C + 7) / 8;
  if (pieces <= 64) return launch<E, F, 64, 1>(a, st);
  if (pieces <= 128) return launch<E, F, 64, 2>(a, st);
  if (pieces <= 256) return launch<E, F, 256, 1>(a, st);
  if (pieces <= 512) return launch<E, F, 256, 2>(a, st);
  if (pieces <= 1024) return launch<E, F, 256, 4>(a, st);
  if (pieces <= 2048) return launch<E, F, 1024, 2>(a, st);
  const unsigned grid = (unsigned)(a->R < 4096 ? a->R : 4096);
  if constexpr (std::is_same<F, Same>::value) {
    hipLaunchKernelGGL(add_rms_norm_any_kernel<E>, dim3(grid), dim3(256), 0, st, *a);
    return sf_check_launch("add_rms_norm_any_kernel");
  } else {
    hipLaunchKernelGGL((add_rms_norm_long_kernel<E, F>), dim3(grid), dim3(256), 0, st, *a);
    return sf_check_launch("add_rms_norm_long_kernel");
  }
}

template <class E>
int launch_type(const sf_add_rms_norm_args* a, bool aligned, hipStream_t st) {
  if (a->codes != nullptr) return a->format == SF_FORMAT_MXFP8 ? launch_rows<E, MxFp8>(a, st) : launch_rows<E, MxFp4>(a, st);
  if (aligned) return launch_rows<E, Same>(a, st);
  hipLaunchKernelGGL(add_rms_norm_any_kernel<E>, dim3((unsigned)(a->R < 4096 ? a->R : 4096)), dim3(256), 0, st, *a);
  return sf_check_launch("add_rms_norm_any_kernel");
}

}  // namespace

extern "C" int sf_hip_add_rms_norm_fwd(const sf_add_rms_norm_args* a, void* stream) {
  if (a == nullptr) { sf_set_error("add rms norm: null args"); return 1; }
  if (a->R < 0 || a->C < 1) { sf_set_error("add rms norm: %lld rows of %d", (long long)a->R, a->C); return 1; }
  if (a->dtype < SF_DTYPE_BF16 || a->dtype > SF_DTYPE_F32) { sf_set_error("add rms norm: element type %d", a->dtype); return 1; }
  if (!(a->eps >= 0.f && a->eps <= 1e30f)) { sf_set_error("add rms norm: eps %g is not finite and >= 0, or above 1e30", (double)a->eps); return 1; }
  if (a->R == 0) return 0;
  if (a->x == nullptr || (a->codes == nullptr) == (a->y == nullptr) || (a->codes != nullptr && a->scales == nullptr)) {
    sf_set_error("add rms norm: x, and either y or codes and scales, must be non-null"); return 1;
  }
  const int size = a->dtype == SF_DTYPE_F32 ? 4 : 2;
  const bool aligned = a->C % 8 == 0 && al16(a->x) && a->x_rs * size % 16 == 0 &&
                       (a->residual == nullptr || (al16(a->residual) && a->r_rs * size % 16 == 0)) &&
                       (a->sum == nullptr || (al16(a->sum) && a->h_rs * size % 16 == 0)) &&
                       (a->y == nullptr || (al16(a->y) && a->y_rs * size % 16 == 0));
  if (a->codes != nullptr) {
    if (a->format != SF_FORMAT_MXFP8 && a->format != SF_FORMAT_MXFP4) { sf_set_error("add rms norm: format %d", a->format); return 1; }
    if (a->C % 32 != 0 || !aligned || !al16(a->codes) || a->c_rs % 16 != 0) {
      sf_set_error("add rms norm: microscaled rows are a multiple of 32 and 16-byte aligned"); return 1;
    }
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case SF_DTYPE_BF16: return launch_type<RowBf16>(a, aligned, st);
    case SF_DTYPE_F16: return launch_type<RowFp16>(a, aligned, st);
    default: return launch_type<RowFp32>(a, aligned, st);
  }
}
