"""Attention over packed sequences against its definition in 64 bits.

Tolerance, element by element, with u = finfo.eps / 2 of the element type, A = sum p |v| / sum p and d the
largest error of a logit: a weight is off by u (its rounding for the product with v) and d, so the
weighted mean by 2 (u + d) A, and its own rounding adds u |o|.  d: the fp32 product of D terms, its
scaling, subtraction and exp2 are off by at most (D + 8) 2^-24 times the sum of |q||k| scale plus the
logit's size.  An fp16 weight below 2^-14 (the largest of its slice is at least 1) is off by 2^-25 at
most: n 2^-25 max |v| in the mean.  fp32 sums of n terms: n 2^-24 A.
"""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def offsets(lens):
  return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


def definition(q, k, v, causal, scale):
  """One sequence in 64 bits on the CPU: (result, tolerance)."""
  dtype = q.dtype
  n, H, D = q.shape
  m, Hk = k.shape[0], k.shape[1]
  u = torch.finfo(dtype).eps / 2
  if n == 0 or m == 0:
    return torch.zeros(n, H, D, dtype=torch.float64), torch.full((n, H, D), 1e-30, dtype=torch.float64)
  q, k, v = (t.detach().cpu().double() for t in (q, k, v))
  g = H // Hk
  k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
  s = scale * torch.einsum("nhd,mhd->hnm", q, k)
  seen = torch.ones(n, m, dtype=torch.bool)
  if causal:
    seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
  s = s.masked_fill(~seen, -math.inf)
  p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
  o = torch.einsum("hnm,mhd->nhd", p, v)
  a = torch.einsum("hnm,mhd->nhd", p, v.abs())
  size = abs(scale) * torch.einsum("nhd,mhd->hnm", q.abs(), k.abs())
  d = (D + 8) * 2.0 ** -24 * 2 * size.masked_fill(~seen, 0).amax(-1).transpose(0, 1)[..., None]
  tol = 2 * (u + d + m * 2.0 ** -24) * a + u * o.abs()
  if dtype == torch.float16:
    tol = tol + m * 2.0 ** -25 * v.abs().amax()
  return o, tol + 1e-30


def check(out, q, k, v, lens_q, lens_k, causal=False, scale=None, starts_k=None):
  scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
  out = out.cpu().double()
  aq = ak = 0
  for b, (n, m) in enumerate(zip(lens_q, lens_k)):
    if starts_k is not None:
      ak = starts_k[b]
    want, tol = definition(q[aq:aq + n], k[ak:ak + m], v[ak:ak + m], causal, scale)
    off = (out[aq:aq + n] - want).abs()
    assert torch.isfinite(out[aq:aq + n]).all(), f"sequence {b}"
    worst = (off / tol).max().item() if n else 0.0
    assert worst <= 1.0, f"sequence {b} ({n} x {m}): error {worst:.2f} of the tolerance"
    aq, ak = aq + n, ak + m


def make(lens_q, lens_k, H, Hk, D, dtype, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda t, h: torch.randn(t, h, D, generator=g).to(dtype).to(DEV)
  return r(sum(lens_q), H), r(sum(lens_k), Hk), r(sum(lens_k), Hk)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 96, 112, 120, 128])
def test_head_dims(D, causal, dtype):
  lens = [70, 1, 33]
  q, k, v = make(lens, lens, 4, 2, D, TYPES[dtype], D)
  check(ops.packed_attention(q, k, v, offsets(lens), causal=causal), q, k, v, lens, lens, causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (6, 2), (8, 8), (5, 1), (33, 1), (40, 8)])
def test_head_groups(heads, causal):
  lens = [130, 64, 5, 129]
  q, k, v = make(lens, lens, *heads, 64, torch.bfloat16, heads[0])
  check(ops.packed_attention(q, k, v, offsets(lens), causal=causal), q, k, v, lens, lens, causal)


LENGTHS = [([1], [1]), ([2], [1]), ([0, 3, 0], [4, 0, 0]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [127, 128, 129]),
           ([255, 257], [256, 255]), ([1, 1, 1, 1], [1, 65, 1000, 0]), ([5], [700]), ([700], [5]), ([300, 2], [1100, 3]),
           ([1] * 70, [(7 * i) % 90 for i in range(70)])]


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("bf16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS, ids=lambda l: "x".join(str(sum(x)) for x in l))
def test_lengths(lens, causal, dtype, D):
  lens_q, lens_k = lens
  q, k, v = make(lens_q, lens_k, 4, 2, D, TYPES[dtype], 5)
  out = ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal)
  check(out, q, k, v, lens_q, lens_k, causal)


@pytest.mark.parametrize("dtype,D,n,m", [("bf16", 128, 1, 9001), ("fp16", 64, 3, 5000), ("bf16", 48, 2, 3300), ("bf16", 96, 1, 2050),
                                         ("bf16", 128, 200, 6000), ("fp16", 32, 333, 4097)])
def test_key_slices(dtype, D, n, m):
  """Few rows and many keys: the workgroups take slices of the keys."""
  q, k, v = make([n], [m], 8, 2, D, TYPES[dtype], m)
  out = ops.packed_attention(q, k, v, offsets([n]), offsets([m]), causal=True)
  check(out, q, k, v, [n], [m], True)
  assert torch.equal(out, ops.packed_attention(q, k, v, offsets([n]), offsets([m]), causal=True))


@pytest.mark.parametrize("dtype,D,lens,heads,causal", [("bf16", 128, [4100], (32, 8), True), ("fp16", 96, [1100, 2300, 7, 1500], (48, 24), False),
                                                       ("bf16", 80, [5000, 3333], (24, 6), True)])
def test_long_rows(dtype, D, lens, heads, causal):
  """Enough long rows for the widest tiles; every 97th row and the last ones."""
  H, Hk = heads
  q, k, v = make(lens, lens, H, Hk, D, TYPES[dtype], D)
  out = ops.packed_attention(q, k, v, offsets(lens), causal=causal)
  assert torch.isfinite(out.float()).all()
  at = 0
  for n in lens:
    rows = torch.tensor(sorted(set(range(0, n, 97)) | set(range(max(n - 40, 0), n))))
    for h in range(0, H, 5):
      kk, vv = k[at:at + n, h // (H // Hk)][:, None], v[at:at + n, h // (H // Hk)][:, None]
      for r in rows.split(64):
        # the sampled rows one by one as sequences of one query over the keys they see
        s = (q[at + r.to(DEV), h].double() @ kk[:, 0].double().T) / math.sqrt(D)
        seen = torch.arange(n, device=DEV)[None] <= r.to(DEV)[:, None] if causal else torch.ones(len(r), n, dtype=torch.bool, device=DEV)
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        want, a = p @ vv[:, 0].double(), p @ vv[:, 0].double().abs()
        u = torch.finfo(TYPES[dtype]).eps / 2
        size = (q[at + r.to(DEV), h].double().abs() @ kk[:, 0].double().abs().T / math.sqrt(D)).amax(-1, keepdim=True)
        tol = 2 * (u + (D + 8) * 2.0 ** -23 * size + n * 2.0 ** -24) * a + u * want.abs()
        if dtype == "fp16":
          tol = tol + n * 2.0 ** -25 * vv.double().abs().amax()
        assert ((out[at + r.to(DEV), h].double() - want).abs() <= tol).all()
    at += n


@pytest.mark.parametrize("n", [1, 40, 300])
def test_caches_with_free_rows(n):
  """Keys in caches of 600 rows each, the free rows NaN; queries of a padded batch."""
  used, room, B = [600, 1, 0, 77, 320], 600, 5
  lens_q = [n, 1, min(n, 3), n // 2, n]
  q, k, v = make([n] * B, [room] * B, 6, 3, 64, torch.bfloat16, n)
  for b, m in enumerate(used):
    k[b * room + m:(b + 1) * room] = math.nan
    v[b * room + m:(b + 1) * room] = math.nan
  for b, m in enumerate(lens_q):
    q[b * n + m:(b + 1) * n] = math.nan
  out = torch.full_like(q, 7.0)
  i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
  got = ops.packed_attention(q, k, v, offsets([n] * B), offsets([room] * B), len_q=i32(lens_q), len_k=i32(used), causal=True, out=out)
  assert got is out
  for b in range(B):
    rows, free = out[b * n:b * n + lens_q[b]], out[b * n + lens_q[b]:(b + 1) * n]
    assert (free == 7.0).all()                     # rows of no sequence are left as they were
    check(rows, q[b * n:b * n + lens_q[b]], k[b * room:b * room + used[b]], v[b * room:b * room + used[b]],
          [lens_q[b]], [used[b]], True)


def test_rows_outside_the_sequences_stay():
  lens = [20, 40]
  q, k, v = make([100], [100], 4, 4, 32, torch.bfloat16)
  out = torch.full_like(q, -3.0)
  cu = torch.tensor([10, 30, 70], dtype=torch.int32, device=DEV)
  ops.packed_attention(q, k, v, cu, out=out)
  assert (out[:10] == -3.0).all() and (out[70:] == -3.0).all()
  check(out[10:70], q[10:70], k[10:70], v[10:70], lens, lens)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,D", [(50, 128), (150, 64), (300, 32)])
def test_later_keys_have_no_influence(n, D, bad):
  """Causal: whatever the keys and values from position p on hold, earlier rows do not change."""
  p = n - 21
  q, k, v = make([n], [n], 4, 2, D, torch.bfloat16, n)
  dirty_k, dirty_v = k.clone(), v.clone()
  dirty_k[p:] = bad
  dirty_v[p::2] = bad
  cu = offsets([n])
  out = ops.packed_attention(q, dirty_k, dirty_v, cu, causal=True)
  # rows before p see clean keys only: their sequence cut off at p
  check(out[:p], q[:p], k[:p], v[:p], [p], [p], True)


@pytest.mark.parametrize("n,D", [(20, 64), (200, 64), (2000, 128)])
def test_values_that_are_not_finite_everywhere(n, D):
  """NaN or infinite in one dim of all values: that dim alone, with the value it has."""
  q, k, v = make([n], [n], 4, 2, D, torch.bfloat16, n)
  clean = ops.packed_attention(q, k, v, offsets([n]), causal=True)
  for bad in (math.nan, math.inf, -math.inf):
    dirty = v.clone()
    dirty[..., 5] = bad
    out = ops.packed_attention(q, k, dirty, offsets([n]), causal=True)
    assert torch.equal(out[..., 5].float().cpu(), torch.full((n, 4), bad)) or (bad != bad and torch.isnan(out[..., 5].float()).all())
    rest = [d for d in range(D) if d != 5]
    # (rows done again are summed in another order)
    u = 2.0 ** -8
    assert ((out[..., rest] - clean[..., rest]).float().abs() <= 6 * u * v.float().abs().amax()).all()


def test_nothing_but_nan():
  q, k, v = make([4000], [4000], 8, 8, 64, torch.bfloat16)
  assert torch.isnan(ops.packed_attention(q, k, torch.full_like(v, math.nan), offsets([4000]), causal=True).float()).all()
  assert torch.isnan(ops.packed_attention(torch.full_like(q, math.nan), k, v, offsets([4000]), causal=True).float()).all()


def test_later_values_have_no_influence_over_key_slices():
  n, m, p = 5, 4000, 3998
  q, k, v = make([n], [m], 2, 1, 128, torch.bfloat16)
  v[p:] = math.inf
  out = ops.packed_attention(q, k, v, offsets([n]), offsets([m]), causal=True)
  clean = n - (m - p)                                # rows that see no key from p on
  check(out[:clean], q[:clean], k[:p], v[:p], [clean], [p], True)
  assert not torch.isfinite(out[clean:].float()).any()


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0, 1e-30])
def test_scales(scale):
  lens = [90, 3, 200]
  q, k, v = make(lens, lens, 2, 1, 32, torch.bfloat16, 8)
  q, k = q / 4, k / 4
  for causal in (False, True):
    check(ops.packed_attention(q, k, v, offsets(lens), causal=causal, scale=scale), q, k, v, lens, lens, causal, scale)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 200])
def test_growing_and_falling_logits(n, dtype):
  """Logits that rise or fall by thousands along the keys: the reference point has to follow, and
  what was summed before it moved weighs nothing."""
  D, m = 64, 900
  q, k, v = make([n], [m], 4, 2, D, TYPES[dtype], 3)
  for sign in (1.0, -1.0):
    ramp = (torch.arange(m, device=DEV, dtype=torch.float32) * sign / 16).to(q.dtype)
    k2, q2 = k.clone(), q.clone()
    k2[..., 0] = ramp[:, None]
    q2[..., 0] = 64.0
    check(ops.packed_attention(q2, k2, v, offsets([n]), offsets([m])), q2, k2, v, [n], [m])


def test_products_past_any_reference_point():
  """Products of 1e30 and 1e36: the largest logit takes all the weight, nothing overflows."""
  n, D = 70, 32
  q, k, v = make([n], [n], 2, 2, D, torch.bfloat16, 4)
  for big in (1e15, 1e18):
    q2, k2 = torch.zeros_like(q), torch.zeros_like(k)
    q2[..., 0] = big
    k2[..., 0] = (torch.arange(n, device=DEV) * 0.25 - 8).to(k.dtype)[:, None] * big    # (exact steps of a quarter)
    out = ops.packed_attention(q2, k2, v, offsets([n]), causal=True).float()
    best = v[torch.arange(n, device=DEV)]                          # the last key seen is the largest
    assert torch.equal(out, best.float())


def test_infinite_logits_of_a_row_give_nan():
  q, k, v = make([4], [4], 1, 1, 32, torch.bfloat16)
  k[:, :, 0] = -math.inf
  q[:, :, 0] = 1.0
  assert torch.isnan(ops.packed_attention(q, k, v, offsets([4])).float()).all()
  k[2:, :, 0] = 0.5
  out = ops.packed_attention(q, k, v, offsets([4]))
  check(out, q, k[2:], v[2:], [4], [2])


@pytest.mark.parametrize("layout", ["fused", "head_major", "shared_heads", "shifted", "wide_last"])
@pytest.mark.parametrize("lens", [[45, 100, 7], [1, 1, 1]])
def test_strides(layout, lens):
  T, H, D = sum(lens), 4, 64
  g = torch.Generator().manual_seed(1)
  r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)
  if layout == "fused":
    x = r(T, 3 * H, D)
    q, k, v = x[:, :H], x[:, H:2 * H], x[:, 2 * H:]
  elif layout == "head_major":
    q, k, v = (r(H, T, D).transpose(0, 1) for _ in range(3))
  elif layout == "shared_heads":
    q, k, v = r(T, H, D), r(T, 1, D).expand(T, H, D), r(T, 1, D).expand(T, H, D)
  elif layout == "shifted":
    q, k, v = (r(T * H * D + 3)[3:].view(T, H, D) for _ in range(3))
  else:
    q, k, v = (r(T, H, 2 * D)[..., ::2] for _ in range(3))
  out = torch.zeros(T, H, 2 * D, dtype=torch.bfloat16, device=DEV)[..., D:]
  for o in (None, out):
    check(ops.packed_attention(q, k, v, offsets(lens), causal=True, out=o), q, k, v, lens, lens, True)


def test_single_rows_of_odd_strides():
  """Torch leaves the strides of single rows and heads arbitrary."""
  x = torch.randn(3, 1, 64).to(torch.bfloat16).to(DEV)
  q, k, v = (x[i].as_strided((1, 1, 64), (1, 3, 1)) for i in range(3))
  assert torch.equal(ops.packed_attention(q, k, v, offsets([1])), v)


def test_offsets_past_32_bits():
  """A cache of more than 2^31 elements, its last sequence and its last rows."""
  rows, Hk, D, n = (1 << 31) // 1024 + 5000, 8, 128, 3000
  k = torch.empty(rows, Hk, D, dtype=torch.bfloat16, device=DEV)
  v = torch.empty(rows, Hk, D, dtype=torch.bfloat16, device=DEV)
  k[-n:] = torch.randn(n, Hk, D, device=DEV).to(k.dtype)
  v[-n:] = torch.randn(n, Hk, D, device=DEV).to(k.dtype)
  q = torch.randn(2, 8, D, device=DEV).to(k.dtype)
  cu_k = torch.tensor([rows - n, rows - 1000, rows], dtype=torch.int32, device=DEV)
  out = ops.packed_attention(q, k, v, offsets([1, 1]), cu_k, causal=True)
  check(out, q, k[-n:], v[-n:], [1, 1], [n - 1000, 1000], True)


def test_wrong_offsets_stay_inside_the_tensors():
  """Negative, decreasing and too large offsets are clamped: sequences they empty have no keys."""
  q, k, v = make([64], [64], 2, 2, 32, torch.bfloat16)
  cu = torch.tensor([-5, 40, 1 << 30, 30, 64], dtype=torch.int32, device=DEV)
  out = ops.packed_attention(q, k, v, cu, torch.tensor([0, 64, 64, 64, 1 << 30], dtype=torch.int32, device=DEV))
  check(out[:30], q[:30], k, v, [30], [64])          # rows of one valid sequence only


@pytest.mark.parametrize("n,m", [([1] * 4, [500, 3, 4000, 129]), ([128, 60, 1, 11], [128, 60, 1, 11])])
def test_capture_and_replay(n, m):
  """A captured call follows the inputs and the lengths that its buffers hold at each replay."""
  q, k, v = make(n, m, 8, 2, 128, torch.bfloat16, 1)
  cu_q, cu_k = offsets(n), offsets(m)
  ops.packed_attention(q, k, v, cu_q, cu_k, causal=True)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      out = ops.packed_attention(q, k, v, cu_q, cu_k, causal=True)
      second = ops.packed_attention(q, k, v, cu_q, cu_k, scale=0.05)
  for step in range(3):
    q.copy_(torch.randn_like(q))
    lens = list(m) if step != 1 else [m[0] - 1] + [m[1] + 1] + list(m[2:])
    if step == 1:
      cu_k.copy_(offsets(lens))
    else:
      cu_k.copy_(offsets(m))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.packed_attention(q, k, v, cu_q, cu_k, causal=True))
    assert torch.equal(second, ops.packed_attention(q, k, v, cu_q, cu_k, scale=0.05))
    check(out, q, k, v, n, lens, True)


def test_other_streams_at_once():
  """Two calls with key slices on two streams: each has its own workspace."""
  a, b = torch.cuda.Stream(), torch.cuda.Stream()
  sets = [make([1], [6000], 8, 2, 128, torch.bfloat16, s) for s in (1, 2)]
  cu_q, cu_k = offsets([1]), offsets([6000])
  torch.cuda.synchronize()
  outs = []
  for _ in range(5):
    for st, (q, k, v) in zip((a, b), sets):
      with torch.cuda.stream(st):
        outs.append(ops.packed_attention(q, k, v, cu_q, cu_k, causal=True))
  torch.cuda.synchronize()
  for i, out in enumerate(outs):
    q, k, v = sets[i % 2]
    check(out, q, k, v, [1], [6000], True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens_q,lens_k", [([300, 65, 513], [300, 65, 513]), ([70, 200], [961, 449]), ([450, 90], [600, 10]), ([129], [4100])])
def test_groups_of_waves_that_share_the_keys(lens_q, lens_k, causal, D, dtype):
  """Few workgroups: odd and even numbers of key tiles, fewer keys than queries, waves without rows, slices besides."""
  q, k, v = make(lens_q, lens_k, 4, 2, D, TYPES[dtype], D)
  if causal:
    v[sum(lens_k) - 1] = math.inf                    # the last key, which only the last query sees
  out = ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal)
  if causal:
    assert not torch.isfinite(out[-1].float()).any()
    out[-1], v[-1] = 0.0, 0.0
    check(out[:-1], q[:-1], k[:-1], v[:-1], lens_q[:-1] + [lens_q[-1] - 1], lens_k[:-1] + [lens_k[-1] - 1], True)
  else:
    check(out, q, k, v, lens_q, lens_k)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("bf16", 24)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sequences,heads", [(2, (16, 2)), (7, (8, 2)), (30, (8, 1)), (64, (3, 1)), (65, (16, 8)), (256, (4, 4))])
def test_slices_by_keys(sequences, heads, causal, dtype, D):
  """Few rows over caches of very different lengths: long ones are split into many slices, short ones into none."""
  g = torch.Generator().manual_seed(sequences)
  lens_k = [(0, 1, 130, 513, 2500, 9000)[i] for i in torch.randint(0, 6, (sequences,), generator=g)]
  lens_k[-1], lens_k[0] = 5000, 77
  lens_q = [(0, 1, 1, 2, 5)[i] for i in torch.randint(0, 5, (sequences,), generator=g)]
  lens_q[0], lens_q[-1] = 9, 1
  q, k, v = make(lens_q, lens_k, *heads, D, TYPES[dtype], D)
  if causal:                                         # what only hidden keys hold
    end = sum(lens_k) - 1
    v[77 - 1], v[end] = math.nan, 3.0
  out = ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal)
  if causal:                                         # the last query of the first sequence sees the NaN
    assert torch.isnan(out[8]).all()
    out[8], v[77 - 1] = 0.0, 0.0
    lens = [8] + lens_q[1:]
    check(torch.cat([out[:8], out[9:]]), torch.cat([q[:8], q[9:]]), k, v, lens, [76] + lens_k[1:], True,
          starts_k=[0] + [sum(lens_k[:b]) for b in range(1, sequences)])
  else:
    check(out, q, k, v, lens_q, lens_k)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sequences,top", [(192, 30), (193, 30), (300, 400), (4097, 20), (9000, 3)])
def test_many_sequences(sequences, top, causal):
  """Beyond 192 sequences a launch of its own counts their tiles; empty ones, a few long ones, lengths in use."""
  g = torch.Generator().manual_seed(sequences)
  room = torch.randint(0, top + 1, (sequences,), generator=g)
  room[::7], room[5], room[-1] = 0, 300, 1
  used = (torch.rand(sequences, generator=g) * (room + 1)).int().clamp(max=room.int())
  q, k, v = make(room.tolist(), room.tolist(), 2, 1, 32, torch.bfloat16, top)
  cu, n = offsets(room.tolist()), used.to(DEV)
  out = torch.full_like(q, 7.0)
  assert ops.packed_attention(q, k, v, cu, causal=causal, out=out) is out
  every = range(sequences) if sequences <= 300 else list(range(0, sequences, 97)) + [5, 6, sequences - 1]
  starts = [0] + room.cumsum(0).tolist()
  for b in every:
    rows = slice(starts[b], starts[b + 1])
    check(out[rows], q[rows], k[rows], v[rows], [room[b].item()], [room[b].item()], causal)
  out.fill_(7.0)
  ops.packed_attention(q, k, v, cu, len_q=n, causal=causal, out=out)
  free = torch.ones(len(q), dtype=torch.bool)
  for b in range(sequences):
    free[starts[b]:starts[b] + used[b]] = False
  assert (out[free.to(DEV)] == 7.0).all()
  for b in every:
    rows = slice(starts[b], starts[b] + used[b])
    check(out[rows], q[rows], k[rows], v[rows], [used[b].item()], [used[b].item()], causal)


def test_many_wrong_offsets():
  """Overlapping, decreasing and too large ones, more tiles than the launch has: no access outside."""
  q, k, v = make([64], [64], 2, 2, 32, torch.bfloat16)
  cu = torch.tensor([0, 1 << 30, -1] * 200 + [10, 64], dtype=torch.int32, device=DEV)
  room = torch.full((192, 2, 32), 7.0, dtype=torch.bfloat16, device=DEV)
  ops.packed_attention(q, k, v, cu, torch.full_like(cu, 64).index_fill_(0, torch.zeros(1, dtype=torch.long, device=DEV), 0), out=room[64:128])
  assert (room[:64] == 7.0).all() and (room[128:] == 7.0).all()
  # a row belongs to several sequences, only the first of them with keys: its result, or zeros
  got, (want, tol) = room[64:128].cpu().double(), definition(q, k, v, False, 1 / math.sqrt(32))
  assert (((got - want).abs() <= tol) | (got == 0)).all()


def test_empty_batch():
  q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
  assert ops.packed_attention(q, q, q, offsets([0, 0])).shape == (0, 4, 64)
  k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
  q = torch.randn(3, 4, 64, device=DEV).to(torch.bfloat16)
  assert (ops.packed_attention(q, k, k, offsets([3]), offsets([0])) == 0).all()


def test_agrees_with_the_padded_attention():
  """The same call as a batch of equal lengths through the framework's padded attention."""
  from sparsefold_amd.backends.hip.attention import dot_product_attention
  B, L, H, D = 3, 150, 4, 48
  q, k, v = make([B * L], [B * L], H, H, D, torch.bfloat16, 2)
  packed = ops.packed_attention(q, k, v, offsets([L] * B))
  padded = dot_product_attention(*(t.view(B, L, H, D) for t in (q, k, v)))
  # both within the tolerance of the definition: at most twice that apart
  for b in range(B):
    s = slice(b * L, (b + 1) * L)
    want, tol = definition(q[s], k[s], v[s], False, D ** -0.5)
    assert ((packed[s] - padded[b]).cpu().double().abs() <= 2 * tol).all()
