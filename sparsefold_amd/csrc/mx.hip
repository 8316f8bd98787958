// Microscaled numbers: codes and scales of rows, and back.
#include "mx.h"

namespace {

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A thread takes 8 elements a step, a quad of lanes a block of 32.  Bound by memory: 16384 x 4096 bf16 to 4 bits 33 us (5.2 TB/s), back
// 26.5.
template <class E, class F>
__global__ __launch_bounds__(256) void mx_encode_kernel(const sf_mx_convert_args a, const uint32_t per_row, const int64_t all) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row);
    Raw8<E> raw;
    raw.load((const typename E::T*)a.x + r * a.x_rs + 8 * (int64_t)c);
    float x[8];
    raw.get(x);
    uint32_t byte;
    const typename F::Codes codes = mx_encode<F>(x, byte);
    *reinterpret_cast<typename F::Codes*>((uint8_t*)a.codes + r * a.c_rs + (int64_t)F::kBytes * c) = codes;
    if ((c & 3) == 0) ((uint8_t*)a.scales)[r * a.s_rs + (c >> 2)] = (uint8_t)byte;
  }
}

template <class E, class F>
__global__ __launch_bounds__(256) void mx_decode_kernel(const sf_mx_convert_args a, const uint32_t per_row, const int64_t all) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row);
    const typename F::Codes codes = *reinterpret_cast<const typename F::Codes*>((const uint8_t*)a.codes + r * a.c_rs + (int64_t)F::kBytes * c);
    const float scale = mx_scale(((const uint8_t*)a.scales)[r * a.s_rs + (c >> 2)]);
    float x[8];
    F::decode(codes, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= scale;
    Raw8<E>::store((typename E::T*)a.x + r * a.x_rs + 8 * (int64_t)c, x);
  }
}

template <class E, class F>
int launch(const sf_mx_convert_args* a, bool encode, hipStream_t st) {
  const uint32_t per_row = (uint32_t)(a->K / 8);
  const int64_t all = a->R * per_row;
  // (whole quads of lanes work on a block: 256 threads a step, blocks of 4)
  const unsigned grid = (unsigned)(all <= 256ll * 16384 ? (all + 255) / 256 : 16384);
  if (encode) hipLaunchKernelGGL((mx_encode_kernel<E, F>), dim3(grid), dim3(256), 0, st, *a, per_row, all);
  else hipLaunchKernelGGL((mx_decode_kernel<E, F>), dim3(grid), dim3(256), 0, st, *a, per_row, all);
  return sf_check_launch(encode ? "mx_encode_kernel" : "mx_decode_kernel");
}

template <class E>
int launch_type(const sf_mx_convert_args* a, bool encode, hipStream_t st) {
  return a->format == SF_FORMAT_MXFP8 ? launch<E, MxFp8>(a, encode, st) : launch<E, MxFp4>(a, encode, st);
}

int convert(const sf_mx_convert_args* a, bool encode, void* stream) {
  if (a == nullptr) { sf_set_error("microscaled: null args"); return 1; }
  if (a->R < 0 || a->K < 32 || a->K % 32 != 0) { sf_set_error("microscaled: rows of %d, a multiple of 32 from 32 on", a->K); return 1; }
  if (a->format != SF_FORMAT_MXFP8 && a->format != SF_FORMAT_MXFP4) { sf_set_error("microscaled: format %d", a->format); return 1; }
  if (a->dtype < SF_DTYPE_BF16 || a->dtype > SF_DTYPE_F32) { sf_set_error("microscaled: element type %d", a->dtype); return 1; }
  if (a->R == 0) return 0;
  const int size = a->dtype == SF_DTYPE_F32 ? 4 : 2;
  if (a->x == nullptr || a->codes == nullptr || a->scales == nullptr) { sf_set_error("microscaled: x, codes and scales must be non-null"); return 1; }
  if (!al16(a->x) || !al16(a->codes) || a->x_rs * size % 16 != 0 || a->c_rs % 16 != 0) {
    sf_set_error("microscaled: rows of x and codes must be 16-byte aligned"); return 1;
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case SF_DTYPE_BF16: return launch_type<RowBf16>(a, encode, st);
    case SF_DTYPE_F16: return launch_type<RowFp16>(a, encode, st);
    default: return launch_type<RowFp32>(a, encode, st);
  }
}

}  // namespace

extern "C" int sf_hip_mx_encode_fwd(const sf_mx_convert_args* a, void* stream) { return convert(a, true, stream); }
extern "C" int sf_hip_mx_decode_fwd(const sf_mx_convert_args* a, void* stream) { return convert(a, false, stream); }
