// A paged cache of keys and values: new rows into their pages, and the attention of new tokens over it (the kernels of
// packed.h, whose tiles find their rows through the table).
#include "packed.h"

namespace {

constexpr char kWhat[] = "paged attention", kWrite[] = "paged write";

// What attention and write ask of the cache alike.
template <class A>
int check_cache(const A* a, const int64_t (&ks)[3], const int64_t (&vs)[3], const void* k, const void* v, const char* what) {
  if (a->pages < 1 || a->pages > INT32_MAX || a->table_cols < 1 || a->page_rows < 16 || a->page_rows % 16 != 0 ||
      (int64_t)a->table_cols * a->page_rows > 1 << 30) {
    sf_set_error("%s: %lld pages of %d rows (a multiple of 16), %d a sequence (2^30 rows at most)", what, (long long)a->pages, a->page_rows,
                 a->table_cols);
    return 1;
  }
  if (k == nullptr || v == nullptr || a->table == nullptr || a->len_k == nullptr) {
    sf_set_error("%s: pages, table and len_k must be non-null", what); return 1;
  }
  if (!aligned16(k) || !aligned16(v)) { sf_set_error("%s: pages must be 16-byte aligned", what); return 1; }
  for (const int64_t* st : {ks, vs})
    if (st[0] < 0 || st[0] % 8 || st[1] % 8 || st[2] % 8 || st[1] < a->D || st[1] >= 1 << 24) {
      sf_set_error("%s: strides of pages must be multiples of 8 elements, of rows in [D, 2^24)", what); return 1;
    }
  return 0;
}

int check(const sf_paged_attention_args* a) {
  if (check_sizes(a, kWhat) || check_cache(a, a->k_s, a->v_s, a->k, a->v, kWhat)) return 1;
  const int G = a->H / a->Hkv;
  if (a->Tq > (1 << 30) / G) {
    sf_set_error("paged attention: %lld queries of %d heads a key head exceed 2^30", (long long)a->Tq, G); return 1;
  }
  if ((a->Tq > 0 && (a->q == nullptr || a->out == nullptr)) || a->cu_q == nullptr) {
    sf_set_error("paged attention: q, out and cu_q must be non-null"); return 1;
  }
  if (!aligned16(a->q) || !aligned16(a->out)) { sf_set_error("paged attention: q and out must be 16-byte aligned"); return 1; }
  for (int i = 0; i < 2; ++i)
    if (a->q_s[i] % 8 || a->o_s[i] % 8) { sf_set_error("paged attention: strides must be multiples of 8 elements"); return 1; }
  return 0;
}

int plan(const sf_paged_attention_args* a, PagedArgs& p, Route& r) {     // (of checked arguments, Tq > 0)
  static_cast<sf_paged_attention_args&>(p) = *a;
  p.div = page_div((uint32_t)a->page_rows >> 4);
  const int64_t most = (int64_t)a->table_cols * a->page_rows;
  return route(&p, a->max_keys > 0 && a->max_keys < most ? a->max_keys : most, r, kWhat);
}

// The last of n + 1 offsets that is at most t (0 where none is): lanes look at 64 of them a step.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n, int t) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool at = lane * step < n && cu[b + min(lane * step, n - 1)] <= t;
    const int skip = max(__popcll(__ballot(at)) - 1, 0) * step;
    b += skip;
    n = min(step, n - skip);
  }
  return b;
}

// A wave takes one row, in turns where it has more than 64 pieces, or as many narrow ones as sf_hip_paged_write_fwd says.  Bound by
// latency (64 tokens of 8 heads of 128 2.7 us) and, from some MB on, by memory (6959 tokens 10.8 us, 5.3 TB/s).
__global__ __launch_bounds__(256) void paged_write_kernel(const sf_paged_write_args a, const int log_rows) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = a.D / 8, pieces = a.Hkv * per;              // 16-byte pieces of a row
  const int64_t t0 = ((int64_t)workgroup() * 4 + wave) << log_rows;
  const int lanes = 64 >> log_rows, mine = lane / lanes;
  char* kd = nullptr;
  char* vd = nullptr;
#pragma unroll 1
  for (int r = 0; r < 1 << log_rows; ++r) {
    const int64_t t = t0 + r;                                // (uniform)
    if (t >= a.T) break;
    const int b = sequence_of(a.cu, a.B, (int)t);
    const int64_t first = a.cu[b], end = min((int64_t)a.cu[b + 1], a.T);
    const int64_t n = a.len_new != nullptr ? min((int64_t)a.len_new[b], end - first) : end - first;
    const int64_t i = t - first, at = (int64_t)a.len_k[b] - n + i;
    if (i < 0 || i >= n || at < 0 || at >= (int64_t)a.table_cols * a.page_rows) continue;
    const int page = (int)(at / a.page_rows), row = (int)(at - (int64_t)page * a.page_rows);
    const int id = a.table[b * a.table_s + page];
    if ((uint32_t)id >= (uint64_t)a.pages) continue;
    if (mine == r) {
      kd = (char*)((uint16_t*)a.k_pages + id * a.kp_s[0] + row * a.kp_s[1]);
      vd = (char*)((uint16_t*)a.v_pages + id * a.vp_s[0] + row * a.vp_s[1]);
    }
  }
  if (kd == nullptr) return;
  const char* const ks = (const char*)((const uint16_t*)a.k + (t0 + mine) * a.k_s[0]);
  const char* const vs = (const char*)((const uint16_t*)a.v + (t0 + mine) * a.v_s[0]);
  for (int p = lane % lanes; p < pieces; p += lanes) {
    const int h = p / per, d = 16 * (p - h * per);
    const u32x4 kx = ld16(ks + 2 * h * a.k_s[1] + d), vx = ld16(vs + 2 * h * a.v_s[1] + d);
    st16(kd + 2 * h * a.kp_s[2] + d, kx);
    st16(vd + 2 * h * a.vp_s[2] + d, vx);
  }
}

}  // namespace

extern "C" size_t sf_hip_paged_attention_workspace_bytes(const sf_paged_attention_args* a) {
  Route r;
  PagedArgs p;
  if (a == nullptr || a->Tq == 0 || check(a) || plan(a, p, r)) return 0;
  return part_bytes(&p, r);
}

extern "C" int sf_hip_paged_attention_fwd(const sf_paged_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (a == nullptr) { sf_set_error("paged attention: null args"); return 1; }
  Route r;
  PagedArgs p;
  if (check(a)) return 1;
  if (a->Tq == 0) return 0;                                  // nothing to write
  if (plan(a, p, r)) return 1;
  return run(&p, r, workspace, workspace_bytes, stream, kWhat);
}

extern "C" int sf_hip_paged_write_fwd(const sf_paged_write_args* a, void* stream) {
  if (a == nullptr) { sf_set_error("paged write: null args"); return 1; }
  if (a->B <= 0 || a->Hkv <= 0 || a->D <= 0 || a->D % 8 != 0 || a->T < 0 || a->T > 1 << 30 || (int64_t)a->Hkv * a->D > 1 << 24) {
    sf_set_error("paged write: B=%d Hkv=%d D=%d (a multiple of 8) T=%lld", a->B, a->Hkv, a->D, (long long)a->T); return 1;
  }
  if (check_cache(a, a->kp_s, a->vp_s, a->k_pages, a->v_pages, kWrite)) return 1;
  if (a->T == 0) return 0;
  if (a->k == nullptr || a->v == nullptr || a->cu == nullptr || !aligned16(a->k) || !aligned16(a->v)) {
    sf_set_error("paged write: k, v and cu must be non-null, k and v 16-byte aligned"); return 1;
  }
  for (int i = 0; i < 2; ++i)
    if (a->k_s[i] % 8 || a->v_s[i] % 8) { sf_set_error("paged write: strides must be multiples of 8 elements"); return 1; }
  // A row a wave up to 8192, which the chip runs at once: a wave's rows are found one after another.  Beyond, up to four that its lanes
  // hold at 16 bytes each (us with 1 / 2 / 4 / up to 16 rows a wave: 64 tokens of 1 head of 32 3.0 / 3.4 / 4.5 / 11.2, 8192 5.3 / 5.0 / 5.4 / 11.6,
  // 16384 8.0 / 7.4 / 7.5 / 11.8, 65536 25.4 / 22.1 / 21.0 / 22.9, 262144 93 / 77 / 70 / 69; of 128 64 tokens 2.8 / 3.3 / 4.5, 8192 5.5 / 5.3 / 5.8, 65536
  // 26.5 / 22.9 / 21.5).
  const int pieces = a->Hkv * (a->D / 8), most = a->T <= 8192 ? 0 : 2;
  int log_rows = 0;
  while (log_rows < most && pieces << (log_rows + 1) <= 64) ++log_rows;
  const int64_t rows = 4ll << log_rows, wgs = (a->T + rows - 1) / rows;          // (up to 2^28)
  const dim3 grid = wgs <= kGridX ? dim3((unsigned)wgs) : dim3(kGridX, (unsigned)((wgs + kGridX - 1) / kGridX));
  hipLaunchKernelGGL(paged_write_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), *a, log_rows);
  return sf_check_launch("paged_write_kernel");
}
