// y = x w^T + bias of 4-bit microscaled operands on large grids, gfx950: tiles of 256 x 256 by 4 waves, one per SIMD, wave tiles of 128 x 128
// with their 256 sums a lane in accumulation registers, persistent.
//
// Per step of 128 k (64 bytes a row) a wave issues 32 matrix instructions back to back in one block, and between them its reads of the
// next step's operands from LDS and its copies of the step after the next three: nothing waits but the block's end, where the
// reads have long returned.  One barrier a step.  Wave tiles of 128 x 128 read 2/3 of the LDS bytes of 128 x 64 ones, and no wave waits
// for another's reads.
//   step t: copies of step t + 1 landed (vmcnt, issue order), barrier, block: products of t, reads of t + 1, copies of t + 4
// The copies of step t + 4 overwrite the stage of step t, whose reads ended (lgkmcnt(0)) in the block before the barrier.
// LDS, scales and results as in the kernel of 8 waves (rows of 64 bytes, pieces XORed by (row / 4) % 4; scales 16 a copy, four
// buffers; whole lines stored by buffer stores).
#include <algorithm>
#include <type_traits>

#include "mx.h"
#include "mx_linear.h"

namespace {

typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint32_t lds_u32;
constexpr int kTile = 256;

template <int N>
__device__ __forceinline__ void wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// A lane's part of the wave's copies: 4 KB of x and of w a step, scales of 64 rows of each.
struct Copies {
  const char *x, *w, *sx, *sw;                               // uniform bases
  uint32_t xo[4], wo[4], sxo, swo;                           // lane offsets
};
struct Operands {
  u32x4 x[2][4], w[2][4];                                    // [64 k][32 rows]
  uint32_t sx[4], sw[4];                                     // words of the rows' scales
};

#define M(C, W, X, V, U, SEL) "v_mfma_scale_f32_32x32x64_f8f6f4 %[" C "], %[" W "], %[" X "], %[" C "], %[" V "], %[" U "] op_sel_hi:" SEL " cbsz:4 blgp:4\n\t"
#define M0(I, J) M("c" #I #J, "w0" #I, "x0" #J, "v" #I, "u" #J, "[0,0,0]")
#define M1(I, J) M("c" #I #J, "w1" #I, "x1" #J, "v" #I, "u" #J, "[1,1,0]")
#define RX(K, J, OFF) "ds_read_b128 %[nx" #K #J "], %[xr" #K "] offset:" #OFF "\n\t"
#define RW(K, J, OFF) "ds_read_b128 %[nw" #K #J "], %[wr" #K "] offset:" #OFF "\n\t"
#define RU(J, OFF) "ds_read_b32 %[nu" #J "], %[ur] offset:" #OFF "\n\t"
#define RV(J, OFF) "ds_read_b32 %[nv" #J "], %[vr] offset:" #OFF "\n\t"
#define SETM(R) "s_mov_b32 m0, %[" R "]\n\t"
#define ADDM "s_add_u32 m0, m0, 0x400\n\t"
#define CP(V, S) "global_load_lds_dwordx4 %[" V "], %[" S "]\n\t"
// The copies of a step at the places C0 .. C15 between the products (m0 a place ahead), those of scales at S.
#define BLOCK(S, C0, C1, C2, C3, C4, C5, C6, C7, C8, C9, C10, C11, C12, C13, C14, C15)                                                     \
  "s_nop 1\n\t" M0(0, 0) RX(0, 0, 0) RU(0, 0) M0(1, 0) RX(0, 1, 2048) RU(1, 512) M0(2, 0) RX(0, 2, 4096) RU(2, 1024) M0(3, 0)                 \
      RX(0, 3, 6144) RU(3, 1536) M0(0, 1) RW(0, 0, 0) RV(0, 0) M0(1, 1) RW(0, 1, 2048) RV(1, 512) M0(2, 1) RW(0, 2, 4096) RV(2, 1024)        \
          M0(3, 1) RW(0, 3, 6144) RV(3, 1536) M0(0, 2) RX(1, 0, 0) M0(1, 2) RX(1, 1, 2048) M0(2, 2) RX(1, 2, 4096) M0(3, 2) RX(1, 3, 6144)   \
              S M0(0, 3) RW(1, 0, 0) M0(1, 3) RW(1, 1, 2048) M0(2, 3) RW(1, 2, 4096) M0(3, 3) RW(1, 3, 6144) M1(0, 0) C0 M1(1, 0) C1         \
                  M1(2, 0) C2 M1(3, 0) C3 M1(0, 1) C4 M1(1, 1) C5 M1(2, 1) C6 M1(3, 1) C7 M1(0, 2) C8 M1(1, 2) C9 M1(2, 2) C10 M1(3, 2) C11  \
                      M1(0, 3) C12 M1(1, 3) C13 M1(2, 3) C14 M1(3, 3) C15 LAST "s_waitcnt lgkmcnt(0)"
// Behind a tile's last step the results are read: 18 wait states after the last product, which the compiler, blind to what a block holds,
// would not keep.  (Between blocks nothing reads them.)
#define LAST "s_cmp_lg_u32 %[more], 0\n\ts_cbranch_scc1 .Lnot_last_%=\n\ts_nop 15\n\ts_nop 7\n\t.Lnot_last_%=:\n\t"
#define CODES SETM("mx"), CP("xo0", "xa"), ADDM, CP("xo1", "xa"), ADDM, CP("xo2", "xa"), ADDM, CP("xo3", "xa"), SETM("mw"), CP("wo0", "wa"), ADDM, \
              CP("wo1", "wa"), ADDM, CP("wo2", "wa"), ADDM, CP("wo3", "wa")
// (jumped over where the step brings no scales: a branch within the block, so that the sums keep their registers)
#define SCALES "s_cmp_eq_u32 %[ms], 0\n\ts_cbranch_scc1 .Lno_scales_%=\n\t" SETM("ms") "s_nop 0\n\t" CP("so", "sa") \
               "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\t" CP("to", "ta") ".Lno_scales_%=:\n\t"
#define EXPAND(...) BLOCK(__VA_ARGS__)
#define ACC(I, J) [c##I##J] "+a"(acc[I][J])
#define OUTX(K, J) [nx##K##J] "=&v"(n.x[K][J])
#define OUTW(K, J) [nw##K##J] "=&v"(n.w[K][J])
#define INX(K, J) [x##K##J] "v"(o.x[K][J])
#define INW(K, J) [w##K##J] "v"(o.w[K][J])
#define RUN(...)                                                                                                                            \
  asm volatile(EXPAND(__VA_ARGS__)                                                                                                          \
               : ACC(0, 0), ACC(0, 1), ACC(0, 2), ACC(0, 3), ACC(1, 0), ACC(1, 1), ACC(1, 2), ACC(1, 3), ACC(2, 0), ACC(2, 1), ACC(2, 2),     \
                 ACC(2, 3), ACC(3, 0), ACC(3, 1), ACC(3, 2), ACC(3, 3), OUTX(0, 0), OUTX(0, 1), OUTX(0, 2), OUTX(0, 3), OUTX(1, 0),           \
                 OUTX(1, 1), OUTX(1, 2), OUTX(1, 3), OUTW(0, 0), OUTW(0, 1), OUTW(0, 2), OUTW(0, 3), OUTW(1, 0), OUTW(1, 1), OUTW(1, 2),      \
                 OUTW(1, 3), [nu0] "=&v"(n.sx[0]), [nu1] "=&v"(n.sx[1]), [nu2] "=&v"(n.sx[2]), [nu3] "=&v"(n.sx[3]), [nv0] "=&v"(n.sw[0]),     \
                 [nv1] "=&v"(n.sw[1]), [nv2] "=&v"(n.sw[2]), [nv3] "=&v"(n.sw[3])                                                           \
               : INX(0, 0), INX(0, 1), INX(0, 2), INX(0, 3), INX(1, 0), INX(1, 1), INX(1, 2), INX(1, 3), INW(0, 0), INW(0, 1), INW(0, 2),     \
                 INW(0, 3), INW(1, 0), INW(1, 1), INW(1, 2), INW(1, 3), [u0] "v"(u[0]), [u1] "v"(u[1]), [u2] "v"(u[2]), [u3] "v"(u[3]),       \
                 [v0] "v"(v[0]), [v1] "v"(v[1]), [v2] "v"(v[2]), [v3] "v"(v[3]), [xr0] "v"(xr), [xr1] "v"(xr ^ 32u), [wr0] "v"(wr),           \
                 [wr1] "v"(wr ^ 32u), [ur] "v"(ur), [vr] "v"(vr), [mx] "s"(mx), [mw] "s"(mw), [ms] "s"(ms), [more] "s"(more), [xa] "s"(xa), [wa] "s"(wa),      \
                 [sa] "s"(sa), [ta] "s"(ta), [xo0] "v"(c.xo[0]), [xo1] "v"(c.xo[1]), [xo2] "v"(c.xo[2]), [xo3] "v"(c.xo[3]),                 \
                 [wo0] "v"(c.wo[0]), [wo1] "v"(c.wo[1]), [wo2] "v"(c.wo[2]), [wo3] "v"(c.wo[3]), [so] "v"(c.sxo), [to] "v"(c.swo)             \
               : "memory", "m0", "scc")

// Products of the step in o, reads of the next one into n, copies of a later one (ms = 0: without scales); more: steps of the tile behind this one.  (The scales' shifts, vector
// instructions, lie two wait states before the products that take them.)
__device__ __forceinline__ void block(f32x16v (&acc)[4][4], const Operands& o, Operands& n, uint32_t xr, uint32_t wr, uint32_t ur, uint32_t vr,
                                      uint32_t mx, uint32_t mw, uint32_t ms, int more, const char* xa, const char* wa, const char* sa,
                                      const char* ta, const Copies& c) {
  const int half = (threadIdx.x >> 5) & 1;
  uint32_t u[4], v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[i] = o.sx[i] >> (8 * half);                            // bytes 0 and 2: the row's blocks of this half
    v[i] = o.sw[i] >> (8 * half);
  }
  RUN(SCALES, CODES);
}
#undef M
#undef M0
#undef M1
#undef RX
#undef RW
#undef RU
#undef RV
#undef SETM
#undef ADDM
#undef CP
#undef BLOCK
#undef CODES
#undef LAST
#undef SCALES
#undef EXPAND
#undef ACC
#undef OUTX
#undef OUTW
#undef INX
#undef INW
#undef RUN

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

template <class E>
__global__ __launch_bounds__(256, 1) void mx_linear_w4_kernel(const sf_mx_linear_args a, const int gx, const int gy, const int total) {
  constexpr int S = 4, CPW = 8, GS = 4;                       // stages, copies of codes a wave and step, steps of a group of scales
  constexpr int XBYTES = kTile * 64, STAGE = 2 * XBYTES, SCALES = 2 * kTile * 16;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STAGE + 4 * SCALES];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, li = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
  // (tiles to XCDs in bands, as in the kernel of 8 waves)
  constexpr int kBand = 5;
  const int per = (total + 7) >> 3, xcd = blockIdx.x & 7, G8 = gridDim.x >> 3;
  const int tend = min(total, (xcd + 1) * per);
  int tile = xcd * per + (int)(blockIdx.x >> 3);
  if (tile >= tend) return;                                   // uniform over the workgroup
  const auto place = [&](int t, int& bx, int& by) __attribute__((always_inline)) {
    const int band = t / (kBand * gy), q = t - band * kBand * gy;
    const int bh = min(kBand, gx - band * kBand);
    by = q / bh;
    bx = band * kBand + q - by * bh;
  };
  // Rows past the end read the last row (their results are not stored).
  const auto sources = [&](int t, Copies& c) __attribute__((always_inline)) {
    int bx, by;
    place(t, bx, by);
    const int64_t m0 = (int64_t)bx * kTile, n0 = (int64_t)by * kTile;
    const int lastx = (int)min(a.M - 1 - m0, (int64_t)kTile - 1), lastw = (int)min((int64_t)a.N - 1 - n0, (int64_t)kTile - 1);
    c.x = (const char*)a.x + m0 * a.x_rs;
    c.w = (const char*)a.w + n0 * a.w_rs;
    c.sx = (const char*)a.x_scales + m0 * a.xs_rs;
    c.sw = (const char*)a.w_scales + n0 * a.ws_rs;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 16 * (4 * wave + u) + (lane >> 2), piece = (lane & 3) ^ ((row >> 2) & 3);
      c.xo[u] = (uint32_t)min(row, lastx) * (uint32_t)a.x_rs + piece * 16;
      c.wo[u] = (uint32_t)min(row, lastw) * (uint32_t)a.w_rs + piece * 16;
    }
    c.sxo = (uint32_t)min(64 * wave + lane, lastx) * (uint32_t)a.xs_rs;
    c.swo = (uint32_t)min(64 * wave + lane, lastw) * (uint32_t)a.ws_rs;
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u32*)smem;
  const uint32_t in_row = (uint32_t)((half ^ ((li >> 2) & 3)) << 4);
  const uint32_t xbase = lds0 + (uint32_t)((wm * 128 + li) * 64) + in_row, wbase = lds0 + XBYTES + (uint32_t)((wn * 128 + li) * 64) + in_row;
  const uint32_t ubase = lds0 + S * STAGE + (wm * 128 + li) * 16, vbase = lds0 + S * STAGE + (kTile + wn * 128 + li) * 16;
  const auto barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  const int n = a.K / 128;                                    // >= S and even (host rule)
  const int blocks = a.K / 32, groups = (n + GS - 1) / GS;
  const auto group_at = [&](int g) __attribute__((always_inline)) { return min(16 * g, blocks - 16); };
  Copies c;
  sources(tile, c);
  __builtin_amdgcn_global_load_lds(c.sx + c.sxo, (lds_u32*)(smem + S * STAGE + wave * 1024), 16, 0, 0);
  __builtin_amdgcn_global_load_lds(c.sw + c.swo, (lds_u32*)(smem + S * STAGE + 4096 + wave * 1024), 16, 0, 0);
#pragma unroll
  for (int t = 0; t < S; ++t) {
    uint8_t* const st = smem + t * STAGE;
#pragma unroll
    for (int u = 0; u < 4; ++u) __builtin_amdgcn_global_load_lds(c.x + (c.xo[u] + t * 64), (lds_u32*)(st + (4 * wave + u) * 1024), 16, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u) __builtin_amdgcn_global_load_lds(c.w + (c.wo[u] + t * 64), (lds_u32*)(st + XBYTES + (4 * wave + u) * 1024), 16, 0, 0);
  }
  wait<(S - 1) * CPW>();
  barrier();
  Operands A, B;
  {
    // step 0, read in one block with its wait
#define R(D, AD, OFF) "ds_read_b128 %" #D ", %[" AD "] offset:" #OFF "\n\t"
    asm volatile(R(0, "x0", 0) R(1, "x0", 2048) R(2, "x0", 4096) R(3, "x0", 6144) R(4, "x1", 0) R(5, "x1", 2048) R(6, "x1", 4096) R(7, "x1", 6144)
                 R(8, "w0", 0) R(9, "w0", 2048) R(10, "w0", 4096) R(11, "w0", 6144) R(12, "w1", 0) R(13, "w1", 2048) R(14, "w1", 4096) R(15, "w1", 6144)
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(A.x[0][0]), "=&v"(A.x[0][1]), "=&v"(A.x[0][2]), "=&v"(A.x[0][3]), "=&v"(A.x[1][0]), "=&v"(A.x[1][1]), "=&v"(A.x[1][2]),
                   "=&v"(A.x[1][3]), "=&v"(A.w[0][0]), "=&v"(A.w[0][1]), "=&v"(A.w[0][2]), "=&v"(A.w[0][3]), "=&v"(A.w[1][0]), "=&v"(A.w[1][1]),
                   "=&v"(A.w[1][2]), "=&v"(A.w[1][3])
                 : [x0] "v"(xbase), [x1] "v"(xbase ^ 32u), [w0] "v"(wbase), [w1] "v"(wbase ^ 32u) : "memory");
#undef R
    asm volatile("ds_read_b32 %0, %8\n\tds_read_b32 %1, %8 offset:512\n\tds_read_b32 %2, %8 offset:1024\n\tds_read_b32 %3, %8 offset:1536\n\t"
                 "ds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:512\n\tds_read_b32 %6, %9 offset:1024\n\tds_read_b32 %7, %9 offset:1536\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(A.sx[0]), "=&v"(A.sx[1]), "=&v"(A.sx[2]), "=&v"(A.sx[3]), "=&v"(A.sw[0]), "=&v"(A.sw[1]), "=&v"(A.sw[2]), "=&v"(A.sw[3])
                 : "v"(ubase), "v"(vbase) : "memory");
  }
  // The stores of a tile's results sit in the memory counter behind the copies of the next tile's step 3: the waits of its first
  // three steps leave them in flight.
  constexpr int kStores = 32;
  bool stored = false;
  int T = 0, G = 0;                                           // steps and groups of scales done: stage (T + t) % S, buffer (G + g) % 4
  f32x16v acc[4][4];                                          // [columns][rows]
  for (;;) {
    const int next = tile + G8;
    const bool has_next = next < tend;                        // uniform
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const auto step = [&](int t, const Operands& o, Operands& nx) __attribute__((always_inline)) {
      // the copies of step t + 1 landed; those of steps t + 2 and t + 3 may stay in flight
      if (stored && t < S - 1) wait<2 * CPW + kStores>();
      else wait<2 * CPW>();
      barrier();
      const int rt = t + 1 < n ? t + 1 : 0;                   // the step read: of this tile or the next
      const int rg = rt / GS;
      const uint32_t so = (uint32_t)((T + t + 1) & (S - 1)) * STAGE;
      const uint32_t sc = (uint32_t)((G + rg + (t + 1 < n ? 0 : groups)) & 3) * SCALES + (4 * rt - group_at(rg));
      const uint32_t to = lds0 + (uint32_t)((T + t) & (S - 1)) * STAGE;      // of step t + S
      const bool own = t + S < n;
      const int ct = own ? t + S : t + S - n, cg = ct / GS;
      const uint32_t ms = ct % GS == 0 ? lds0 + S * STAGE + (uint32_t)((G + cg + (own ? 0 : groups)) & 3) * SCALES + wave * 1024 : 0;
      const char *const xa = c.x + (int64_t)ct * 64, *const wa = c.w + (int64_t)ct * 64, *const sa = c.sx + group_at(cg), *const ta = c.sw + group_at(cg);
      block(acc, o, nx, xbase + so, wbase + so, ubase + sc, vbase + sc, to + wave * 4096, to + XBYTES + wave * 4096, ms, n - 1 - t, xa, wa, sa, ta, c);
    };
    for (int t = 0; t < n; t += 2) {
      // from here on the copies are the next tile's (without one this one's first steps again, so that every step has its copies)
      if (t + S == n) sources(has_next ? next : tile, c);
      step(t, A, B);
      step(t + 1, B, A);
    }
    T += n;
    G += groups;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+a"(acc[i][j]));

    // ---- results of this wave's 128 x 128: lane (row li, half) has columns 8 (r / 4) + 4 half + r % 4 ----
    {
      int bx, by;
      place(tile, bx, by);
      const int64_t m0 = (int64_t)bx * kTile + wm * 128;
      const int64_t rows = a.M - m0;
      uint32_t line = 2 * (uint32_t)a.y_rs;                   // (taken up here: kept over the loop, the rows' offsets cost registers)
      int own_row = li & ~3, own_col = 16 * (lane & 3) + 8 * half;
      int own_half = 16 * half;
      asm volatile("" : "+s"(line), "+v"(own_row), "+v"(own_col), "+v"(own_half));
      const __amdgpu_buffer_rsrc_t rb =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.bias), (short)0, a.bias != nullptr ? 4 * a.N : 0, 0x00020000);
      const __amdgpu_buffer_rsrc_t r =
          __builtin_amdgcn_make_buffer_rsrc((uint16_t*)a.y + (rows > 0 ? m0 : 0) * a.y_rs, (short)0, rows > 0 ? 0x7fffff00 : 0, 0x00020000);
#pragma unroll
      for (int part = 0; part < 2; ++part) {                  // 64 columns
        const int n0 = by * kTile + wn * 128 + 64 * part;
        f32x4 b[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // (columns past the last read nothing, and neither does a call without a bias)
            const auto w = __builtin_amdgcn_raw_buffer_load_b128(rb, 4 * (n0 + 32 * i + 8 * q) + own_half, 0, 0);
            b[i][q] = __builtin_bit_cast(f32x4, w);
          }
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          u32x4 p[4];                                         // 8 columns 16 c + 8 half .. of row li
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            const f32x16v& v = acc[2 * part + (c4 >> 1)][mb];
            const f32x4 b0 = b[c4 >> 1][2 * (c4 & 1)], b1 = b[c4 >> 1][2 * (c4 & 1) + 1];
            const int q = 8 * (c4 & 1);
            const float lo[8] = {v[q] + b0[0], v[q + 1] + b0[1], v[q + 2] + b0[2], v[q + 3] + b0[3],
                                 v[q + 4] + b1[0], v[q + 5] + b1[1], v[q + 6] + b1[2], v[q + 7] + b1[3]};
            const u32x4 k = E::pack(lo);                      // columns 16 c + 4 half .. + 3 and 8 further
            const uint32_t k0 = k[0], k1 = k[1], k2 = k[2], k3 = k[3];
            const auto y0 = __builtin_amdgcn_permlane32_swap(k0, k2, false, false);
            const auto y1 = __builtin_amdgcn_permlane32_swap(k1, k3, false, false);
            p[c4] = u32x4{y0[0], y1[0], y0[1], y1[1]};
          }
          turn<0xB1>(p[0], p[1], lane & 1);                   // (whole lines a store, as in the kernel of 8 waves)
          turn<0xB1>(p[2], p[3], lane & 1);
          turn<0x4E>(p[0], p[2], lane & 2);
          turn<0x4E>(p[1], p[3], lane & 2);
          const int col = n0 + own_col;
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            const int row = 32 * mb + own_row + c4;
            const uint32_t off = row < rows && col < a.N ? (uint32_t)row * line + 2u * (uint32_t)col : 0x80000000u;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, p[c4]), r, (int)off, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);                  // (registers)
        }
      }
      stored = true;
    }
    if (!has_next) break;
    tile = next;
  }
  wait<0>();                                                  // (no copy outlives the workgroup's LDS)
}

template <class E>
int launch(const sf_mx_linear_args* a, hipStream_t stream) {
  const int64_t gx = (a->M + kTile - 1) / kTile, gy = ((int64_t)a->N + kTile - 1) / kTile, total = gx * gy;
  const int n = std::max(sf_resident_workgroups(reinterpret_cast<const void*>(mx_linear_w4_kernel<E>), 256) / 8 * 8, 8);
  hipLaunchKernelGGL(mx_linear_w4_kernel<E>, dim3((unsigned)std::min<int64_t>(n, (total + 7) / 8 * 8)), dim3(256), 0, stream, *a, (int)gx, (int)gy,
                     (int)total);
  return sf_check_launch("mx_linear_w4_kernel");
}

}  // namespace

bool sf_mx_linear_w4_ok(const sf_mx_linear_args* a) {
  return a->x_format == SF_FORMAT_MXFP4 && a->w_format == SF_FORMAT_MXFP4 && a->K % 256 == 0;     // (an even number of steps)
}

int sf_mx_linear_w4_launch(const sf_mx_linear_args* a, hipStream_t stream) {
  return a->dtype == SF_DTYPE_BF16 ? launch<RowBf16>(a, stream) : launch<RowFp16>(a, stream);
}
