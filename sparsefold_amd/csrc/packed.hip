// Attention over packed sequences, keys and values in rows of one tensor: the kernels of packed.h.
#include "packed.h"

namespace {

constexpr char kWhat[] = "packed attention";

int check(const sf_packed_attention_args* a) {
  if (a->Tk < 0) { sf_set_error("packed attention: %lld keys", (long long)a->Tk); return 1; }
  if (check_sizes(a, kWhat)) return 1;
  const int G = a->H / a->Hkv;
  if (a->Tk > 1 << 30 || a->Tq > (1 << 30) / G) {
    sf_set_error("packed attention: %lld queries of %d heads a key head, or %lld keys, exceed 2^30", (long long)a->Tq, G, (long long)a->Tk);
    return 1;
  }
  if (a->Tq > 0 && (a->q == nullptr || a->out == nullptr || (a->Tk > 0 && (a->k == nullptr || a->v == nullptr)))) {
    sf_set_error("packed attention: q, k, v and out must be non-null"); return 1;
  }
  if (a->cu_q == nullptr || a->cu_k == nullptr) { sf_set_error("packed attention: cu_q and cu_k must be non-null"); return 1; }
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) {
    sf_set_error("packed attention: q, k, v and out must be 16-byte aligned"); return 1;
  }
  for (int i = 0; i < 2; ++i)
    if (a->q_s[i] % 8 || a->k_s[i] % 8 || a->v_s[i] % 8 || a->o_s[i] % 8) {
      sf_set_error("packed attention: strides must be multiples of 8 elements"); return 1;
    }
  for (const int64_t st : {a->k_s[0], a->v_s[0]})
    if (st < a->D || st >= 1 << 24) {
      sf_set_error("packed attention: key and value row strides must lie in [D, 2^24)"); return 1;
    }
  return 0;
}

int64_t keys(const sf_packed_attention_args* a) { return (a->Tk + a->B - 1) / a->B; }      // of an average sequence

}  // namespace

extern "C" size_t sf_hip_packed_attention_workspace_bytes(const sf_packed_attention_args* a) {
  Route r;
  if (a == nullptr || a->Tq == 0 || check(a) || route(a, keys(a), r, kWhat)) return 0;
  return part_bytes(a, r);
}

extern "C" int sf_hip_packed_attention_fwd(const sf_packed_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (a == nullptr) { sf_set_error("packed attention: null args"); return 1; }
  Route r;
  if (a->Tq == 0 && a->B > 0) return 0;                      // nothing to write
  if (check(a) || route(a, keys(a), r, kWhat)) return 1;
  return run(a, r, workspace, workspace_bytes, stream, kWhat);
}
