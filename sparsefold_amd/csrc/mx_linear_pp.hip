// y = x w^T + bias of microscaled operands on large grids, gfx950: tiles of 256 x 256, 8 waves (2 x 4, wave tiles of 128 x 64), two per
// SIMD, through a ring of four LDS stages, persistent.  The schedule is that of the bf16 product on large grids: two groups
// of one wave per SIMD run half a step apart, one reads a step's operands from LDS and copies a later step while the other's
// matrix instructions run; one barrier separates the halves.  Every barrier is met by all waves; the copies of step t + 3
// overwrite the stage of step t - 1, whose last reads ended a barrier before, and a wave's own copies of step t + 1 are
// waited for before the barrier ahead of its first reads.
//
// A step is 64 bytes of a row of x: 64 k of 8 bits, 128 k of 4 bits; w as many k, so 4-bit w beside 8-bit x takes rows of 32
// bytes.  Rows of 64 bytes keep their 16-byte pieces XORed by (row / 4) % 4; of 32 bytes two share a line, slots 2 (row % 2) +
// piece, XORed by (row / 8) % 2: so 16 lanes that read together cover all banks.
// Scales come 16 at a time, 512 k: each wave copies those of 64 rows, into one of four LDS buffers, with the first step that needs
// them, and a lane reads its rows' words with the operands.  (Copied with every step, 2 or 4 bytes a row, they touched 64
// lines an instruction for 256 bytes: 8192^3 took 330 us of 4 bits and 582 of 8.)
// Results are rounded in registers, brought together to whole lines by exchanges between lanes, and stored by buffer stores
// that drop what lies outside, so that their number, which the waits count, does not depend on the tile.
//
// 8192^3: 287 to 315 us of 4 bits, 3.5 to 3.8 PFLOP/s, by the card, and 489 to 515 of 8 bits, 2.25 to 2.13 (products of 8192^3 in bf16: 1.3; matrix
// instructions alone, on random codes in registers: 6.8 and 3.8, clocks held by power).  Over K from 512 to 8192 at 8192 x 8192 a tile takes 6 us
// (9.6 of 8 and 8 bits) and 1.08 us a step of 128 k of 4 bits, 0.92 a step of 64 k of 8 and 8, 0.90 of 8 and 4: the step, not the tile's start
// and end, is 90% of the time.  With all codes zero 236 us of 4 bits and 425 of 8; of 4 bits without the copies 240.  4 waves of 128 x 128, one a
// SIMD, with the next step's reads between the products took as long (283 us, 285 with copies of whole 128-byte lines), so the two
// groups' alternation is not what bounds it; L2 hits 90% of the lines asked for.
#include <algorithm>
#include <type_traits>

#include "index.h"
#include "mx.h"
#include "mx_linear.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint32_t lds_u32;
constexpr int kTile = 256;

template <int N>
__device__ __forceinline__ void wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
// vmcnt(n * CPW), n = the steps that may stay in flight (uniform)
template <int CPW, int MAX>
__device__ __forceinline__ void wait_steps(int n) {
  if (n >= MAX) wait<MAX * CPW>();
  else if constexpr (MAX > 0) wait_steps<CPW, MAX - 1>(n);
}

// The lane's part of a wave's copies: x and w chunks of 1 KB, scales of 64 rows.
struct Copies {
  const char *x, *w, *s;                                     // uniform bases
  uint32_t xo[2], wo[2], so;                                 // lane offsets
};

// The operands of a step and the scales' words of its rows, then -- COPY -- the wave's copies of a later step, then the wait for
// the reads: the copies go out while the reads return.  One block with its wait inside.  mx, mw, ms: LDS addresses of the copies.
#define MX_READS_X "ds_read_b128 %0, %[x0]\n\tds_read_b128 %1, %[x0] offset:2048\n\tds_read_b128 %2, %[x0] offset:4096\n\t" \
                   "ds_read_b128 %3, %[x0] offset:6144\n\tds_read_b128 %4, %[x1]\n\tds_read_b128 %5, %[x1] offset:2048\n\t" \
                   "ds_read_b128 %6, %[x1] offset:4096\n\tds_read_b128 %7, %[x1] offset:6144\n\t"
#define MX_READS_W2 "ds_read_b128 %8, %[w0]\n\tds_read_b128 %9, %[w0] offset:2048\n\tds_read_b128 %10, %[w1]\n\tds_read_b128 %11, %[w1] offset:2048\n\t"
#define MX_READS_W1 "ds_read_b128 %8, %[w0]\n\tds_read_b128 %9, %[w0] offset:1024\n\t"
#define MX_READS_S "ds_read_b32 %[s0], %[sx]\n\tds_read_b32 %[s1], %[sx] offset:512\n\tds_read_b32 %[s2], %[sx] offset:1024\n\t" \
                   "ds_read_b32 %[s3], %[sx] offset:1536\n\tds_read_b32 %[s4], %[sw]\n\tds_read_b32 %[s5], %[sw] offset:512\n\t"
#define MX_COPY_X "s_mov_b32 m0, %[mx]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[xo0], %[xa]\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t" \
                  "global_load_lds_dwordx4 %[xo1], %[xa]\n\t"
#define MX_COPY_W1 "s_mov_b32 m0, %[mw]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[wo0], %[wa]\n\t"
#define MX_COPY_W2 MX_COPY_W1 "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[wo1], %[wa]\n\t"
#define MX_COPY_S "s_mov_b32 m0, %[ms]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[so], %[sa]\n\t"
#define MX_WAIT "s_waitcnt lgkmcnt(0)"
#define MX_OUT_X "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[1][2]), "=&v"(x[1][3])
#define MX_OUT_S [s0] "=&v"(s[0]), [s1] "=&v"(s[1]), [s2] "=&v"(s[2]), [s3] "=&v"(s[3]), [s4] "=&v"(s[4]), [s5] "=&v"(s[5])
#define MX_IN [x0] "v"(x0), [x1] "v"(x0 ^ 32u), [w0] "v"(w0), [w1] "v"(w0 ^ 32u), [sx] "v"(sx), [sw] "v"(sw)
#define MX_IN_COPY [mx] "s"(mx), [mw] "s"(mw), [ms] "s"(ms), [xa] "s"(xa), [wa] "s"(wa), [sa] "s"(sa), [xo0] "v"(c.xo[0]), [xo1] "v"(c.xo[1]), \
                   [wo0] "v"(c.wo[0]), [wo1] "v"(c.wo[1]), [so] "v"(c.so)
enum Copy { kNone, kCodes, kCodesAndScales };
template <int WC, Copy COPY>
__device__ __forceinline__ void read_step(uint32_t x0, uint32_t w0, uint32_t sx, uint32_t sw, u32x4 (&x)[2][4], u32x4 (&w)[2][2], uint32_t (&s)[6],
                                          uint32_t mx, uint32_t mw, uint32_t ms, const char* xa, const char* wa, const char* sa, const Copies& c) {
#define MX_STEP(READS, COPIES, OUT_W) asm volatile(READS COPIES MX_WAIT : MX_OUT_X, OUT_W, MX_OUT_S : MX_IN, MX_IN_COPY : "memory", "m0", "scc")
#define MX_OUT_W1 "=&v"(w[0][0]), "=&v"(w[0][1])
#define MX_OUT_W2 "=&v"(w[0][0]), "=&v"(w[0][1]), "=&v"(w[1][0]), "=&v"(w[1][1])
#define MX_ARGS(...) __VA_ARGS__
  if constexpr (WC == 2) {
    if constexpr (COPY == kCodesAndScales) MX_STEP(MX_READS_X MX_READS_W2 MX_READS_S, MX_COPY_S MX_COPY_X MX_COPY_W2, MX_ARGS(MX_OUT_W2));
    else if constexpr (COPY == kCodes) MX_STEP(MX_READS_X MX_READS_W2 MX_READS_S, MX_COPY_X MX_COPY_W2, MX_ARGS(MX_OUT_W2));
    else MX_STEP(MX_READS_X MX_READS_W2 MX_READS_S, "", MX_ARGS(MX_OUT_W2));
  } else {
    if constexpr (COPY == kCodesAndScales) MX_STEP(MX_READS_X MX_READS_W1 MX_READS_S, MX_COPY_S MX_COPY_X MX_COPY_W1, MX_ARGS(MX_OUT_W1));
    else if constexpr (COPY == kCodes) MX_STEP(MX_READS_X MX_READS_W1 MX_READS_S, MX_COPY_X MX_COPY_W1, MX_ARGS(MX_OUT_W1));
    else MX_STEP(MX_READS_X MX_READS_W1 MX_READS_S, "", MX_ARGS(MX_OUT_W1));
  }
#undef MX_STEP
#undef MX_OUT_W1
#undef MX_OUT_W2
#undef MX_ARGS
}

__device__ __forceinline__ i32x8 join8(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
__device__ __forceinline__ i32x8 join4(u32x4 a) { return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}; }

// Exchanges lo of the lanes with `bit` for hi of their partners without it (DPP: the partner in the quad).
template <int DPP>
__device__ __forceinline__ void turn(u32x4& lo, u32x4& hi, bool bit) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t l = lo[e], h = hi[e];
    const uint32_t from_l = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)l, DPP, 0xF, 0xF, true);
    const uint32_t from_h = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)h, DPP, 0xF, 0xF, true);
    lo[e] = bit ? from_h : l;
    hi[e] = bit ? h : from_l;
  }
}

template <class E, class FX, class FW>
__global__ __launch_bounds__(512) void mx_linear_pp_kernel(const sf_mx_linear_args a, const int gx, const int gy, const int total) {
  constexpr bool x8 = FX::kFormat == SF_FORMAT_MXFP8, w8 = FW::kFormat == SF_FORMAT_MXFP8;
  constexpr int S = 4, A = S - 1;
  constexpr int WROW = x8 && !w8 ? 32 : 64, WC = WROW / 32;   // bytes of a row of w in a step, copies of w a wave
  constexpr int SB = x8 ? 2 : 4;                              // blocks of 32 in a step
  constexpr int GS = 16 / SB;                                 // steps of a group of scales
  constexpr int XBYTES = kTile * 64, WBYTES = kTile * WROW, STAGE = XBYTES + WBYTES, SCALES = 2 * kTile * 16;
  constexpr int CPW = 2 + WC;                                 // (and a copy of scales before those of a group's first step)
  constexpr int MB = 4, NB = 2;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STAGE + 4 * SCALES];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const bool late = wave >= 4;                                // the second wave of each SIMD
  // Each XCD takes a contiguous range of tiles, in bands of 5 tile rows, so that the tiles it runs together form a block of both
  // operands.
  const int G8 = gridDim.x >> 3;
  const TileWalk walk = tiles_on_xcd(blockIdx.x, total);
  const int tend = walk.end;
  int tile = walk.first;
  if (tile >= tend) return;                                   // uniform over the workgroup
  const auto place = [&](int t, int& bx, int& by) __attribute__((always_inline)) { banded_tile<5>(t, gx, gy, bx, by); };
  // Rows past the end read the last row (their results are not stored).
  const auto sources = [&](int t, Copies& c) __attribute__((always_inline)) {
    int bx, by;
    place(t, bx, by);
    const int64_t m0 = (int64_t)bx * kTile, n0 = (int64_t)by * kTile;
    const int lastx = (int)min(a.M - 1 - m0, (int64_t)kTile - 1), lastw = (int)min((int64_t)a.N - 1 - n0, (int64_t)kTile - 1);
    c.x = (const char*)a.x + m0 * a.x_rs;
    c.w = (const char*)a.w + n0 * a.w_rs;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 16 * (2 * wave + u) + (lane >> 2), piece = (lane & 3) ^ ((row >> 2) & 3);
      c.xo[u] = (uint32_t)min(row, lastx) * (uint32_t)a.x_rs + piece * 16;
      if constexpr (WROW == 64) {
        c.wo[u] = (uint32_t)min(row, lastw) * (uint32_t)a.w_rs + piece * 16;
      } else {
        const int line = 16 * wave + (lane >> 2), slot = (lane & 3) ^ ((line >> 2) & 1);
        c.wo[u] = (uint32_t)min(2 * line + (slot >> 1), lastw) * (uint32_t)a.w_rs + (slot & 1) * 16;
      }
    }
    const int srow = 64 * (wave & 3) + lane;
    if (wave < 4) {                                           // (uniform)
      c.s = (const char*)a.x_scales + m0 * a.xs_rs;
      c.so = (uint32_t)min(srow, lastx) * (uint32_t)a.xs_rs;
    } else {
      c.s = (const char*)a.w_scales + n0 * a.ws_rs;
      c.so = (uint32_t)min(srow, lastw) * (uint32_t)a.ws_rs;
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u32*)smem;
  const uint32_t xbase = lds0 + (uint32_t)((wm * 128 + li) * 64 + ((half ^ ((li >> 2) & 3)) << 4));
  const uint32_t wbase = lds0 + XBYTES +
                         (WROW == 64 ? (uint32_t)((wn * 64 + li) * 64 + ((half ^ ((li >> 2) & 3)) << 4))
                                     : (uint32_t)((wn * 32 + (li >> 1)) * 64 + (((2 * (li & 1) + half) ^ ((li >> 3) & 1)) << 4)));
  const uint32_t sxbase = lds0 + S * STAGE + (wm * 128 + li) * 16, swbase = lds0 + S * STAGE + (kTile + wn * 64 + li) * 16;
  const auto barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  const int n = a.K / (32 * SB);                              // >= A (host rule)
  const int blocks = a.K / 32, groups = (n + GS - 1) / GS;
  const auto group_at = [&](int g) __attribute__((always_inline)) { return scales_of_group(g, blocks); };
  Copies c;
  sources(tile, c);
  __builtin_amdgcn_global_load_lds(c.s + c.so, (lds_u32*)(smem + S * STAGE + wave * 1024), 16, 0, 0);
#pragma unroll
  for (int t = 0; t < A; ++t) {
    uint8_t* const st = smem + t * STAGE;
#pragma unroll
    for (int u = 0; u < 2; ++u) __builtin_amdgcn_global_load_lds(c.x + (c.xo[u] + t * 64), (lds_u32*)(st + (2 * wave + u) * 1024), 16, 0, 0);
#pragma unroll
    for (int u = 0; u < WC; ++u)
      __builtin_amdgcn_global_load_lds(c.w + (c.wo[u] + t * WROW), (lds_u32*)(st + XBYTES + (WC * wave + u) * 1024), 16, 0, 0);
  }
  wait<(A - 1) * CPW>();
  barrier();
  if (late) barrier();
  // The stores of a tile's epilogue sit in the memory counter between the copies of the next tile's steps A - 1 and A: the
  // first A - 1 waits of a tile leave them in flight.
  constexpr int kStores = MB * NB * 2;
  bool stored = false;
  int T = 0;                                                  // steps done: the stage of step t is (T + t) % S
  int G = 0;                                                  // groups done: the buffer of group g is (G + g) % 4
  for (;;) {
    const int next = tile + G8;
    const bool has_next = next < tend;                        // uniform
    Copies nc;
    sources(has_next ? next : tile, nc);
    f32x16v acc[MB][NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[mb][nb][r] = 0.f;
    u32x4 xa[2][MB], wa[2][NB];
    uint32_t s[6];
    for (int t = 0; t < n; ++t) {
      const uint32_t so = (uint32_t)((T + t) & A) * STAGE;
      const uint32_t to = lds0 + (uint32_t)((T + t + A) & A) * STAGE;
      const uint32_t mx = to + wave * 2048, mw = to + XBYTES + wave * WC * 1024;
      const int g = t / GS, at = SB * t - group_at(g);        // the step's first scale among its group's
      const uint32_t sc0 = (uint32_t)((G + g) & 3) * SCALES + (at & ~3);
      // read step t; copy step t + A of this tile, or step t + A - n of the next one
      const bool own = t + A < n;                             // (uniform, as all that follows from it)
      const int ct = own ? t + A : t + A - n, cg = ct / GS;
      const bool with_scales = ct % GS == 0;
      const uint32_t ms = lds0 + S * STAGE + (uint32_t)((G + cg + (own ? 0 : groups)) & 3) * SCALES + wave * 1024;
      const Copies& from = own ? c : nc;
      const char *const xf = from.x + (int64_t)ct * 64, *const wf = from.w + (int64_t)ct * WROW, *const sf = from.s + group_at(cg);
      if (own) {
        if (with_scales) read_step<WC, kCodesAndScales>(xbase + so, wbase + so, sxbase + sc0, swbase + sc0, xa, wa, s, mx, mw, ms, xf, wf, sf, c);
        else read_step<WC, kCodes>(xbase + so, wbase + so, sxbase + sc0, swbase + sc0, xa, wa, s, mx, mw, ms, xf, wf, sf, c);
      } else if (has_next) {
        if (with_scales) read_step<WC, kCodesAndScales>(xbase + so, wbase + so, sxbase + sc0, swbase + sc0, xa, wa, s, mx, mw, ms, xf, wf, sf, nc);
        else read_step<WC, kCodes>(xbase + so, wbase + so, sxbase + sc0, swbase + sc0, xa, wa, s, mx, mw, ms, xf, wf, sf, nc);
      } else {
        read_step<WC, kNone>(xbase + so, wbase + so, sxbase + sc0, swbase + sc0, xa, wa, s, mx, mw, ms, xf, wf, sf, c);
      }
      // the copies of step t + 1 have landed (in issue order); those of steps t + 2 .. t + A may stay in flight (left: how many
      // of them exist), and the stores issued between A - 1 and A
      const int left = has_next ? A : n - 2 - t;
      const bool relax = stored && t < A - 1 && left >= A - 1;   // uniform
      const auto landed = [&]() __attribute__((always_inline)) {
        if (relax) wait<(A - 1) * CPW + kStores>();
        else wait_steps<CPW, A - 1>(left);
      };
      if (late) landed();
      barrier();
      uint32_t sc[6];
#pragma unroll
      for (int i = 0; i < 6; ++i) sc[i] = s[i] >> (8 * half + (x8 ? 8 * (at & 2) : 0));
      if constexpr (x8) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8 ? join8(wa[0][nb], wa[1][nb]) : join4(wa[0][nb]), join8(xa[0][mb], xa[1][mb]),
                                                                          acc[mb][nb], w8 ? 0 : 4, 0, 0, (int)sc[4 + nb], 0, (int)sc[mb]);
      } else {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join4(wa[0][nb]), join4(xa[0][mb]), acc[mb][nb], 4, 4, 0, (int)sc[4 + nb],
                                                                          0, (int)sc[mb]);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join4(wa[1][nb]), join4(xa[1][mb]), acc[mb][nb], 4, 4, 2, (int)sc[4 + nb],
                                                                          2, (int)sc[mb]);
      }
      if (!late) landed();
      barrier();
    }
    T += n;
    G += groups;

    // ---- epilogue of this wave's 128 x 64 part: lane (row li, half) has columns 8 (r / 4) + 4 half + r % 4 ----
    {
      int bx, by;
      place(tile, bx, by);
      const int64_t m0 = (int64_t)bx * kTile + wm * 128;
      const int n0 = by * kTile + wn * 64;
      if (a.bias != nullptr) {                                // (uniform; every load comes before the first store)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 b4 = *reinterpret_cast<const f32x4*>(a.bias + min(n0 + 32 * nb + 8 * q + 4 * half, a.N - 4));
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[mb][nb][4 * q + e] += b4[e];
          }
      }
      const int64_t rows = a.M - m0;
      uint32_t line = 2 * (uint32_t)a.y_rs;                   // (taken up here: kept over the loop, the rows' offsets cost registers)
      int own_row = li & ~3, own_col = 16 * (lane & 3) + 8 * half;
      asm volatile("" : "+s"(line), "+v"(own_row), "+v"(own_col));
      const __amdgpu_buffer_rsrc_t r =
          __builtin_amdgcn_make_buffer_rsrc((uint16_t*)a.y + (rows > 0 ? m0 : 0) * a.y_rs, (short)0, rows > 0 ? 0x7fffff00 : 0, 0x00020000);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        u32x4 p[4];                                           // 8 columns 16 c + 8 half .. of row li: c = 2 nb + q
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          const f32x16v& v = acc[mb][c4 >> 1];
          const int q = 8 * (c4 & 1);
          const float lo[8] = {v[q], v[q + 1], v[q + 2], v[q + 3], v[q + 4], v[q + 5], v[q + 6], v[q + 7]};
          const u32x4 k = E::pack(lo);                        // columns 16 c + 4 half .. + 3 and 8 further
          const uint32_t k0 = k[0], k1 = k[1], k2 = k[2], k3 = k[3];
          const auto y0 = __builtin_amdgcn_permlane32_swap(k0, k2, false, false);
          const auto y1 = __builtin_amdgcn_permlane32_swap(k1, k3, false, false);
          p[c4] = u32x4{y0[0], y1[0], y0[1], y1[1]};
        }
        // Four lanes that hold four pieces of a row each turn them over, so that a store takes whole lines: lane 4 i + b's
        // piece c goes to lane 4 i + c's place b.  (32 bytes of each of 32 rows a store: 8192 x 8192 x 1024 of 4 bits 66 us.)
        turn<0xB1>(p[0], p[1], lane & 1);
        turn<0xB1>(p[2], p[3], lane & 1);
        turn<0x4E>(p[0], p[2], lane & 2);
        turn<0x4E>(p[1], p[3], lane & 2);
        const int col = n0 + own_col;
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          const int row = 32 * mb + own_row + c4;
          const uint32_t off = row < rows && col < a.N ? (uint32_t)row * line + 2u * (uint32_t)col : 0x80000000u;
          typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, p[c4]), r, (int)off, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);                    // (registers)
      }
      stored = true;
    }
    if (!has_next) break;
    tile = next;
    c = nc;
  }
  if (!late) barrier();                                       // the late group's extra first barrier
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class E, class FX, class FW>
int launch(const sf_mx_linear_args* a, hipStream_t stream) {
  const int64_t gx = (a->M + kTile - 1) / kTile, gy = ((int64_t)a->N + kTile - 1) / kTile, total = gx * gy;
  const int n = std::max(sf_resident_workgroups(reinterpret_cast<const void*>(mx_linear_pp_kernel<E, FX, FW>), 512) / 8 * 8, 8);
  hipLaunchKernelGGL((mx_linear_pp_kernel<E, FX, FW>), dim3((unsigned)std::min<int64_t>(n, (total + 7) / 8 * 8)), dim3(512), 0, stream, *a, (int)gx,
                     (int)gy, (int)total);
  return sf_check_launch("mx_linear_pp_kernel");
}

template <class E>
int launch_formats(const sf_mx_linear_args* a, hipStream_t st) {
  if (a->x_format == SF_FORMAT_MXFP4) return launch<E, MxFp4, MxFp4>(a, st);
  if (a->w_format == SF_FORMAT_MXFP4) return launch<E, MxFp8, MxFp4>(a, st);
  return launch<E, MxFp8, MxFp8>(a, st);
}

}  // namespace

// What the kernel assumes: whole steps, at least four of them, 16 scales a row and words of them aligned, aligned rows, offsets inside a tile that fit 32 bits; and sizes
// for which its tiles pay.  The rest takes tiles of 128 (8000 x 8000 x 8064, 8 and 8, 8 and 4, 4 and 4 bits: 505, 480, 302 us here; of
// 8096 k 788, 652, 495; 8001 columns 660, 595, 456).
bool sf_mx_linear_pp_ok(const sf_mx_linear_args* a) {
  if (a->K % 128 != 0 || a->K < 512 || a->N % 8 != 0 || a->M < kTile || a->N < kTile) return false;
  if (!al16(a->y) || a->y_rs % 8 != 0 || a->y_rs >= 1 << 22 || (a->bias && !al16(a->bias))) return false;
  if (((uintptr_t)a->x_scales | (uintptr_t)a->w_scales | (uintptr_t)a->xs_rs | (uintptr_t)a->ws_rs) % 4 != 0) return false;
  const int64_t total = ((a->M + kTile - 1) / kTile) * (((int64_t)a->N + kTile - 1) / kTile);
  // (4096 x 4096 weights, 8 and 8 bits: 2048 rows, 128 tiles, 64 us here and 50 in tiles of 128; 2304 63 and 64; 3000 64 and 66; 4096 70 and 87)
  return total >= 160 && total < 1ll << 30;
}

int sf_mx_linear_pp_launch(const sf_mx_linear_args* a, hipStream_t stream) {
  return a->dtype == SF_DTYPE_BF16 ? launch_formats<RowBf16>(a, stream) : launch_formats<RowFp16>(a, stream);
}
