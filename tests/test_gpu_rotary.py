"""Rotary positions and the norm of queries and keys before them, against the definition in 64 bits.

Tolerance, element by element, u = finfo.eps / 2 of the element type, e = 2^-24: the angle's cos and sin
are off by 4 e (its rounding after the reduction and the series), times the magnitude, product and sum
add 4 e more: 8 e (|a| + |b|) |magnitude|.  A norm's fp32 sums of D terms are off by (D + 8) e relative, its
three products by 3 e, a layer norm's difference from the mean by (D + 8) e of the row's largest
value.  One rounding at the end: u |y|.
"""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E24 = 2.0 ** -24


def definition(x, positions, freqs, interleaved=False, magnitude=1.0, norm=None, weight=None, bias=None, eps=1e-6):
  """(result, tolerance) of [T, H, D] in 64 bits."""
  u = torch.finfo(x.dtype).eps / 2
  x = x.detach().cpu().double()
  D, R = x.shape[-1], 2 * freqs.numel()
  slack = torch.zeros_like(x)
  if norm is not None:
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.cpu().double()
    b = torch.zeros(D, dtype=torch.float64) if bias is None else bias.cpu().double()
    if norm == "layer":
      x = x - x.mean(-1, keepdim=True)
      # the mean's error, relative to the largest value of the row
      slack = (D + 8) * E24 * x.abs().amax(-1, keepdim=True).expand_as(x)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    slack = 2 * slack * r * w.abs() + (D + 11) * E24 * (x * r * w).abs() + 2 * E24 * (x * r * w + b).abs()
    x = x * r * w + b
  angle = positions.cpu().double()[:, None, None] * freqs.cpu()
  c, s = angle.cos() * magnitude, angle.sin() * magnitude
  first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
  y, tol = x.clone(), slack.clone()
  a, b = x[..., first], x[..., second]
  y[..., first], y[..., second] = a * c - b * s, b * c + a * s
  turned = 8 * E24 * (a.abs() + b.abs()) * abs(magnitude) + (slack[..., first] + slack[..., second]) * abs(magnitude)
  tol[..., first], tol[..., second] = turned, turned
  return y, tol + u * (y.abs() + tol) + torch.finfo(torch.float32).tiny + (2.0 ** -25 if u == 2.0 ** -11 else 0.0)


def check(got, x, *args, **kw):
  want, tol = definition(x, *args, **kw)
  got = got.cpu().double()
  assert torch.isfinite(got).all()
  worst = ((got - want).abs() / tol).max().item()
  assert worst <= 1.0, f"error {worst:.2f} of the tolerance"


def rand(*shape, dtype=torch.float32, seed=0):
  return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


SIZES = [(1, 2, 1, 2, 2), (3, 5, 2, 10, 4), (7, 4, 4, 24, 24), (9, 16, 4, 32, 16), (5, 3, 1, 40, 40), (6, 2, 2, 48, 24), (65, 8, 2, 64, 64),
         (4, 6, 3, 80, 80), (3, 4, 2, 96, 48), (130, 32, 8, 128, 128), (17, 8, 1, 128, 64), (2, 3, 3, 130, 130), (5, 4, 1, 256, 256),
         (3, 2, 1, 255, 30), (2, 1, 1, 129, 2), (11, 1, 1, 72, 36)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_rotary(size, interleaved, dtype):
  T, H, Hk, D, R = size
  q, k = rand(T, H, D, dtype=TYPES[dtype], seed=D), rand(T, Hk, D, dtype=TYPES[dtype], seed=R)
  pos = torch.arange(100, 100 + T, dtype=torch.int32, device=DEV)
  f = ops.rotary_frequencies(R, device=DEV)
  oq, ok = ops.rotary(q, k, pos, f, interleaved=interleaved, magnitude=1.25)
  check(oq, q, pos, f, interleaved, 1.25)
  check(ok, k, pos, f, interleaved, 1.25)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_qk_norm_rotary(size, norm, dtype):
  T, H, Hk, D, R = size
  q, k = rand(T, H, D, dtype=TYPES[dtype], seed=D) * 3 + 1, rand(T, Hk, D, dtype=TYPES[dtype], seed=R)
  pos = torch.arange(T, dtype=torch.int64, device=DEV) * 17
  f = ops.rotary_frequencies(R, device=DEV)
  qw, kw = 1 + 0.3 * rand(D, seed=1), 1 + 0.3 * rand(D, seed=2)
  qb, kb = (rand(D, seed=3), rand(D, seed=4)) if norm == "layer" else (None, None)
  interleaved = T % 2 == 1
  oq, ok = ops.qk_norm_rotary(q, k, qw, kw, pos, f, norm=norm, q_bias=qb, k_bias=kb, interleaved=interleaved, eps=1e-5)
  check(oq, q, pos, f, interleaved, norm=norm, weight=qw, bias=qb, eps=1e-5)
  check(ok, k, pos, f, interleaved, norm=norm, weight=kw, bias=kb, eps=1e-5)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_without_weights_and_keys(norm):
  q = rand(5, 3, 64, dtype=torch.bfloat16)
  pos, f = torch.arange(5, device=DEV), ops.rotary_frequencies(64, device=DEV)
  oq, ok = ops.qk_norm_rotary(q, None, None, None, pos, f, norm=norm)
  assert ok is None
  check(oq, q, pos, f, norm=norm)
  oq, ok = ops.rotary(q, None, pos, f)
  assert ok is None
  check(oq, q, pos, f)


def test_far_positions():
  """Positions up to 2^40: the angle keeps its digits (64-bit products are off by 2^-53 of 2^40 / 2 pi turns)."""
  pos = torch.tensor([0, 1, -1, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, (1 << 35) + 7, -(1 << 33) - 5], dtype=torch.int64, device=DEV)
  q = rand(8, 2, 64)
  f = ops.rotary_frequencies(64, device=DEV)
  oq, _ = ops.rotary(q, None, pos, f)
  want, tol = definition(q, pos, f)
  # both sides form the angle in 64 bits: each is off by 2^-51 of it at most
  tol = tol + 2 * 2.0 ** -51 * pos.abs().max().item() * 4
  assert ((oq.cpu().double() - want).abs() <= tol).all()


def test_leading_dims_and_broadcast_positions():
  B, L, H, D = 3, 11, 4, 32
  q, k = rand(B, L, H, D, dtype=torch.bfloat16), rand(B, L, 2, D, dtype=torch.bfloat16, seed=1)
  f = ops.rotary_frequencies(16, device=DEV)
  pos = torch.arange(L, dtype=torch.int32, device=DEV)
  oq, ok = ops.rotary(q, k, pos, f)
  assert oq.shape == q.shape and ok.shape == k.shape
  for b in range(B):
    check(oq[b], q[b], pos, f)
    check(ok[b], k[b], pos, f)
  pos2 = torch.randint(0, 1000, (B, L), device=DEV)
  oq, ok = ops.rotary(q, k, pos2, f)
  for b in range(B):
    check(ok[b], k[b], pos2[b], f)


@pytest.mark.parametrize("op", ["rotary", "rms"])
@pytest.mark.parametrize("layout", ["fused", "head_major", "shifted", "wide_last", "odd_rows"])
def test_strides_and_in_place(layout, op):
  T, H, Hk, D = 13, 4, 2, 64
  dtype = torch.bfloat16
  if layout == "fused":
    x = rand(T, H + 2 * Hk, D, dtype=dtype)
    q, k = x[:, :H], x[:, H:H + Hk]
  elif layout == "head_major":
    q, k = rand(H, T, D, dtype=dtype).transpose(0, 1), rand(Hk, T, D, dtype=dtype).transpose(0, 1)
  elif layout == "shifted":
    q, k = rand(T * H * D + 1, dtype=dtype)[1:].view(T, H, D), rand(T * Hk * D + 1, dtype=dtype)[1:].view(T, Hk, D)
  elif layout == "wide_last":
    q, k = rand(T, H, 2 * D, dtype=dtype)[..., ::2], rand(T, Hk, 2 * D, dtype=dtype)[..., ::2]
  else:
    q, k = rand(T, H, D + 5, dtype=dtype)[..., 5:], rand(T, Hk, D + 5, dtype=dtype)[..., :D]
  pos, f = torch.arange(T, device=DEV), ops.rotary_frequencies(D, device=DEV)
  w = 1 + 0.1 * rand(D, seed=5)
  call = (lambda **kw: ops.rotary(q, k, pos, f, **kw)) if op == "rotary" else (lambda **kw: ops.qk_norm_rotary(q, k, w, w, pos, f, **kw))
  how = {} if op == "rotary" else dict(norm="rms", weight=w)
  oq, ok = call()
  check(oq, q, pos, f, **how)
  check(ok, k, pos, f, **how)
  if layout != "wide_last":
    rest = x[:, H + Hk:].clone() if layout == "fused" else None
    iq, ik = call(out_q=q, out_k=k)
    assert iq is q and ik is k and torch.equal(q, oq) and torch.equal(k, ok)
    if rest is not None:
      assert torch.equal(x[:, H + Hk:], rest)


def test_values_that_are_not_finite_stay_in_their_head():
  q = rand(4, 3, 64, dtype=torch.bfloat16)
  q[1, 1, 5] = math.nan
  q[2, 0, 60] = math.inf
  pos, f = torch.arange(4, device=DEV), ops.rotary_frequencies(64, device=DEV)
  for oq, _ in (ops.rotary(q, None, pos, f), ops.qk_norm_rotary(q, None, None, None, pos, f)):
    bad = ~torch.isfinite(oq.float()).all(-1)
    assert bad[1, 1] and bad[2, 0] and bad.sum() == 2


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [(128, 64), (96, 48), (64, 24), (40, 2), (255, 30), (130, 4)], ids=lambda d: "x".join(map(str, d)))
def test_dims_behind_the_rotated_ones_are_copied(dims, interleaved, dtype):
  """Bit for bit, infinities, NaN and negative zeros among them, and the rotated dims know nothing of them."""
  D, R = dims
  q, k = rand(7, 5, D, dtype=TYPES[dtype]), rand(7, 2, D, dtype=TYPES[dtype], seed=1)
  pos, f = torch.arange(7, device=DEV), ops.rotary_frequencies(R, device=DEV)
  want = ops.rotary(q, k, pos, f, interleaved=interleaved, magnitude=1.5)
  for t in (q, k):
    t[::2, :, R::3], t[1::2, :, R + 1::3], t[:, 1:, D - 1] = math.inf, -0.0, -math.inf
    t[3, 0, R:] = math.nan
  got = ops.rotary(q, k, pos, f, interleaved=interleaved, magnitude=1.5)
  for t, w, g in zip((q, k), want, got):
    assert torch.equal(g[..., :R], w[..., :R])
    assert torch.equal(torch.isnan(g[..., R:]), torch.isnan(t[..., R:]))
    assert torch.equal(g[..., R:].nan_to_num(nan=5.0), t[..., R:].nan_to_num(nan=5.0))
    assert torch.equal(torch.signbit(g[..., R:])[~torch.isnan(t[..., R:])], torch.signbit(t[..., R:])[~torch.isnan(t[..., R:])])


def test_a_graph_that_saved_what_is_overwritten_refuses():
  w = torch.ones(64, device=DEV, requires_grad=True)
  q = rand(4, 2, 64)
  y = (q * w).sum()
  ops.rotary(q, None, torch.arange(4, device=DEV), ops.rotary_frequencies(64, device=DEV), out_q=q)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    y.backward()
  with torch.inference_mode():
    q = rand(4, 2, 64)
    ops.rotary(q, None, torch.arange(4, device=DEV), ops.rotary_frequencies(64, device=DEV), out_q=q)


def test_no_tokens():
  q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
  oq, _ = ops.rotary(q, None, torch.empty(0, dtype=torch.int32, device=DEV), ops.rotary_frequencies(64, device=DEV))
  assert oq.shape == (0, 4, 64)


def test_capture_and_replay():
  q, k = rand(9, 8, 128, dtype=torch.bfloat16), rand(9, 2, 128, dtype=torch.bfloat16, seed=1)
  pos, f = torch.arange(9, device=DEV), ops.rotary_frequencies(128, device=DEV)
  w = 1 + 0.1 * rand(128, seed=2)
  ops.qk_norm_rotary(q, k, w, w, pos, f)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    oq, ok = ops.qk_norm_rotary(q, k, w, w, pos, f)
  for _ in range(3):
    q.copy_(torch.randn_like(q))
    pos.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    eq, ek = ops.qk_norm_rotary(q, k, w, w, pos, f)
    assert torch.equal(oq, eq) and torch.equal(ok, ek)


def test_a_layer_of_packed_sequences():
  """Projection, norm with rotation, attention, output projection, as a sequence model runs them: the
  prompt at once against its last tokens one by one over a cache."""
  lens, H, Hk, D, C = [37, 130, 1], 8, 2, 64, 256
  T = sum(lens)
  g = torch.Generator().manual_seed(7)
  bf = torch.bfloat16
  x = torch.randn(T, C, generator=g).to(bf).to(DEV)
  w_in = (torch.randn((H + 2 * Hk) * D, C, generator=g) / math.sqrt(C)).to(bf).to(DEV)
  w_out = (torch.randn(C, H * D, generator=g) / math.sqrt(H * D)).to(bf).to(DEV)
  nq, nk = 1 + 0.1 * rand(D, seed=1), 1 + 0.1 * rand(D, seed=2)
  f = ops.rotary_frequencies(D, scaling="turns", factor=4.0, original_length=2048, device=DEV)
  pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(DEV)
  cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)

  def qkv(rows, positions):
    y = ops.linear(rows, w_in).view(-1, H + 2 * Hk, D)
    q, k = ops.qk_norm_rotary(y[:, :H], y[:, H:H + Hk], nq, nk, positions, f, out_q=y[:, :H], out_k=y[:, H:H + Hk])
    return q, k, y[:, H + Hk:]

  q, k, v = qkv(x, pos)
  att = ops.packed_attention(q, k, v, cu, causal=True)
  out = ops.linear(att.view(T, H * D), w_out, residual=x)
  # against 64 bits, from the rounded projections on
  y = ops.linear(x, w_in).view(-1, H + 2 * Hk, D)
  for b, n in enumerate(lens):
    s = slice(sum(lens[:b]), sum(lens[:b]) + n)
    check(q[s], y[s, :H], pos[s], f, norm="rms", weight=nq)
    check(k[s], y[s, H:H + Hk], pos[s], f, norm="rms", weight=nk)
    qd, kd, vd = (t[s].cpu().double() for t in (q, k, v))
    kd, vd = kd.repeat_interleave(H // Hk, 1), vd.repeat_interleave(H // Hk, 1)
    sc = torch.einsum("nhd,mhd->hnm", qd, kd) / math.sqrt(D)
    sc = sc.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
    p = torch.softmax(sc, -1)
    want = torch.einsum("hnm,mhd->nhd", p, vd)
    bound = 3 * 2.0 ** -8 * torch.einsum("hnm,mhd->nhd", p, vd.abs())     # weights and result rounded, and 64 bits' worth of fp32
    assert ((att[s].cpu().double() - want).abs() <= bound * 1.01 + 1e-6).all()
  assert torch.isfinite(out.float()).all()
  # the last token of each sequence alone, over a cache that holds the others and free rows
  room = 160
  kc = torch.full((len(lens) * room, Hk, D), math.nan, dtype=bf, device=DEV)
  vc = torch.full_like(kc, math.nan)
  last = [sum(lens[:b + 1]) - 1 for b in range(len(lens))]
  for b, n in enumerate(lens):
    kc[b * room:b * room + n - 1] = k[last[b] - n + 1:last[b]]
    vc[b * room:b * room + n - 1] = v[last[b] - n + 1:last[b]]
  q1, k1, v1 = qkv(x[last], pos[last])
  rows = torch.tensor([b * room + n - 1 for b, n in enumerate(lens)], device=DEV)
  kc[rows], vc[rows] = k1, v1
  one = ops.packed_attention(q1, kc, vc, torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV),
                             torch.arange(0, (len(lens) + 1) * room, room, dtype=torch.int32, device=DEV),
                             len_k=torch.tensor(lens, dtype=torch.int32, device=DEV), causal=True)
  scale = v.float().abs().max().item()
  assert ((one - att[last]).float().abs() <= 6 * 2.0 ** -8 * scale).all()   # both sides off by 3 u A, A <= max |v|
