"""Packed attention at the ends of the number range, by every kernel route: logits far from zero whose
differences are exact, values near the largest, weights far below the row's largest.

Logits: products that fp32 holds exactly leave the difference from the row's largest as it is, so a weight is off by
the rounding of difference times scale (differences up to 100 in log2 units: 3 products and sums, 100 * 3 * 2^-24 < 2^-15)
and of exp2 (2^-22): d = 2^-15 in the tolerance 2 (u + d + n 2^-24) A + u |o|, with u = finfo.eps / 2 of the element type and
A = sum p |v|.
"""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops
from tests.test_gpu_packed_attention import DEV, TYPES, check, make, offsets

pytestmark = pytest.mark.gpu

# (queries, keys, heads): shared key slices, stream, tiles of one and two groups of waves, sliced tiles
ROUTES = [(1, 9000, (8, 2)), (9, 300, (8, 2)), (200, 200, (8, 2)), (333, 5000, (8, 2)), (1300, 1300, (32, 32))]

# first two: the second lies at 2^24 log2 units; (digits of q, digits of k, step, scale)
FAR = [((256, 256, 1), (177 * 256, 114, 24), 1, 1.0), ((4096,), (4096,), 2, 1.0), ((4096,), (4096,), 2, -1.0),
       ((16384,), (12288,), 16, 1.0), ((256, 256, 1), (20 * 256, 7, 3), 1, 1.0)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("route", ROUTES, ids=lambda r: f"{r[0]}x{r[1]}")
@pytest.mark.parametrize("far", FAR, ids=lambda f: f"{sum(a * b for a, b in zip(f[0], f[1]))}by{f[2] * f[3]:g}")
def test_logits_far_from_zero(far, route, causal, dtype):
  """Keys a few exact steps apart: every other query row; the rows between have small logits."""
  (n, m, (H, Hk)), (qd, kd, step, scale) = route, far
  D, g = 32, torch.Generator().manual_seed(n)
  dt = TYPES[dtype]
  x = torch.randint(-3, 0, (m,), generator=g).float()
  x[37] = 0.0                                        # one key above all others
  sign = 1.0 if scale > 0 else -1.0
  q, k = torch.zeros(n, H, D), torch.zeros(m, Hk, D)
  for i, (a, b) in enumerate(zip(qd, kd)):
    q[::2, :, i], k[:, :, i] = a, sign * b
  q[::2, :, 8] = 1.0
  k[:, :, 8] = (sign * step * x)[:, None]
  q[1::2, :, 16:] = torch.randn(len(range(1, n, 2)), H, 16, generator=g) / 2
  k[:, :, 16:] = torch.randn(m, Hk, 16, generator=g) / 2
  q, k = q.to(dt).double(), k.to(dt).double()
  v = torch.randn(m, Hk, D, generator=g).to(dt)
  out = ops.packed_attention(q.to(dt).to(DEV), k.to(dt).to(DEV), v.to(DEV), offsets([n]), offsets([m]), causal=causal, scale=scale).cpu().double()
  u, vd = torch.finfo(dt).eps / 2, v.double()
  for h in range(0, H, max(H // 4, 1)):
    s = scale * q[:, h] @ k[:, h // (H // Hk)].T
    if causal:
      s = s.masked_fill(torch.arange(m)[None] > torch.arange(n)[:, None] + (m - n), -math.inf)
    p = torch.softmax(s, -1)
    want, a = p @ vd[:, h // (H // Hk)], p @ vd[:, h // (H // Hk)].abs()
    tol = 2 * (u + 2.0 ** -15 + m * 2.0 ** -24) * a + u * want.abs() + (m * 2.0 ** -25 * vd.abs().amax() if dtype == "fp16" else 0.0)
    worst = ((out[:, h] - want).abs() / tol).amax(-1)
    assert worst.max() <= 1.0, f"head {h}: rows {torch.nonzero(worst > 1).flatten().tolist()[:5]} at {worst.max().item():.2f} of the tolerance"


@pytest.mark.parametrize("kind", ["rising", "largest", "signs", "steep"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("route", ROUTES, ids=lambda r: f"{r[0]}x{r[1]}")
def test_values_near_the_largest(route, D, causal, kind):
  """bf16 values whose sum, or whose product with a weight above 1, passes fp32: the mean does not."""
  n, m, (H, Hk) = route
  q, k, v = make([n], [m], H, Hk, D, torch.bfloat16, 11)
  if kind == "rising":                               # logits 34.7 nats above those of the later keys
    q, k, v = torch.zeros_like(q), torch.zeros_like(k), torch.full_like(v, 2.0 ** 80)
    q[..., 0] = 1.0
    k[:m // 2, :, 0] = 34.75 * math.sqrt(D)
  elif kind == "steep":                              # rising all along, by a nat every 8 keys, over 40 nats
    q[..., 0] = math.sqrt(D)
    k[..., 0] = (40.0 - torch.arange(m, device=DEV) / 8).clamp(min=0).to(k.dtype)[:, None]
    v = v * 2.0 ** 110
  elif kind == "largest":
    q, v = torch.zeros_like(q), torch.full_like(v, torch.finfo(torch.bfloat16).max)
  else:
    v = v.sign() * 2.0 ** 126
  check(ops.packed_attention(q, k, v, offsets([n]), offsets([m]), causal=causal), q, k, v, [n], [m], causal)


@pytest.mark.parametrize("route", ROUTES, ids=lambda r: f"{r[0]}x{r[1]}")
def test_small_values_keep_their_digits(route):
  n, m, (H, Hk) = route
  q, k, v = make([n], [m], H, Hk, 64, torch.bfloat16, 12)
  v = v * 2.0 ** -60
  out = ops.packed_attention(q, k, v, offsets([n]), offsets([m]))
  check(out * 2.0 ** 60, q, k, v * 2.0 ** 60, [n], [m])


@pytest.mark.parametrize("nats", [17.375, 19.0])
def test_fp16_weights_far_below_the_largest(nats):
  """One key above 30000 others whose weights are 2^-25.07 or 2^-27.4 of its: a weight is off by 2^-25 where the largest is
  2^4 2^-1/2 at least, so n 2^-28.5 max |v|, and by 2 u of itself where it is normal."""
  n, m, H, D = 1300, 30000, 32, 32                   # (enough workgroups that all keys share a reference point)
  q, k = torch.zeros(n, H, D, dtype=torch.float16, device=DEV), torch.zeros(m, H, D, dtype=torch.float16, device=DEV)
  v = (1 + torch.rand(m, H, D, generator=torch.Generator().manual_seed(1)) / 4).half().to(DEV)
  q[..., 0], k[-1, :, 0], v[-1] = 1.0, nats, 0.0
  out = ops.packed_attention(q, k, v, offsets([n]), offsets([m]), scale=1.0).double()
  p = math.exp(-nats) / (1 + (m - 1) * math.exp(-nats))
  want = p * v.double().sum(0)
  assert ((out - want).abs() <= m * 2.0 ** -28.5 * 1.25 + 3 * 2.0 ** -11 * want).all()


def test_more_workgroups_than_a_launch_dimension_holds():
  """2^21 sequences of one token, 8 key heads: 2^24 workgroups of 256 threads and some.  One key each: its value."""
  B, H, D = (1 << 21) + 5, 8, 8
  g = torch.Generator(device=DEV).manual_seed(2)
  q, k, v = (torch.randn(B, H, D, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(3))
  cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
  assert torch.equal(ops.packed_attention(q, k, v, cu), v)
  used = torch.ones(B, dtype=torch.int32, device=DEV)
  used[::3] = 0
  out = torch.full_like(q, 7.0)
  ops.packed_attention(q, k, v, cu, len_q=used, out=out)
  assert torch.equal(out[used == 1], v[used == 1]) and (out[::3] == 7.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,share", [(128, 0.02), (64, 0.0005), (24, 0.3)])
@pytest.mark.parametrize("route", ROUTES + [(5, 40, (4, 1)), (4200, 4200, (32, 8))], ids=lambda r: f"{r[0]}x{r[1]}")
def test_values_that_are_not_finite_here_and_there(route, D, share, dtype):
  """Causal, a share of the values NaN or infinite: a result has what its row sees in its dim, and nothing of what it does not."""
  n, m, (H, Hk) = route
  q, k, v = make([n], [m], H, Hk, D, TYPES[dtype], 7)
  q = q / 4                                          # (every weight is far from vanishing)
  kind = torch.rand(m, Hk, D, generator=torch.Generator().manual_seed(m)).to(DEV) / share
  for i, bad in enumerate((math.inf, -math.inf, math.nan)):
    v[(kind >= i / 3) & (kind < (i + 1) / 3)] = bad
  out = ops.packed_attention(q, k, v, offsets([n]), offsets([m]), causal=True)
  some = sorted(set(range(0, n, max(n // 60, 1))) | set(range(max(n - 40, 0), n)))
  for h in range(0, H, max(H // 3, 1)):
    vh, oh = v[:, h // (H // Hk)].cpu().double(), out[some, h].cpu().double()
    s = q[some, h].cpu().double() @ k[:, h // (H // Hk)].cpu().double().T / math.sqrt(D)
    limit = torch.tensor(some) + (m - n)
    p = torch.softmax(s.masked_fill(torch.arange(m)[None] > limit[:, None], -math.inf), -1)
    nan, top, low = (c.double().cumsum(0)[limit] > 0 for c in (torch.isnan(vh), vh == math.inf, vh == -math.inf))
    nan |= top & low
    assert torch.equal(torch.isnan(oh), nan)
    assert torch.equal(oh == math.inf, top & ~nan) and torch.equal(oh == -math.inf, low & ~nan)
    rest = ~(nan | top | low)
    vf = vh.nan_to_num(0.0, 0.0, 0.0)
    want, a, u = p @ vf, p @ vf.abs(), torch.finfo(TYPES[dtype]).eps / 2
    size = (q[some, h].cpu().double().abs() @ k[:, h // (H // Hk)].cpu().double().abs().T).amax() / math.sqrt(D)
    tol = 2 * (u + (D + 8) * 2.0 ** -23 * size + m * 2.0 ** -24) * a + u * want.abs() + (m * 2.0 ** -30 * 4 if dtype == "fp16" else 0.0) + 1e-30
    assert ((oh - want).abs() <= tol)[rest].all()


def sampled(out, q, k, v, causal):
  """Rows of one sequence against the definition, two heads: every 61st, the first and the last ones."""
  (n, H, D), (m, Hk, _), dt = q.shape, k.shape, q.dtype
  some = torch.tensor(sorted(set(range(0, n, 61)) | set(range(min(n, 20))) | set(range(max(n - 40, 0), n))), device=DEV)
  u = torch.finfo(dt).eps / 2
  for h in (0, H - 1):
    qh, kh, vh = q[some, h].double(), k[:, h // (H // Hk)].double(), v[:, h // (H // Hk)].double()
    s, size = qh @ kh.T / math.sqrt(D), (qh.abs() @ kh.abs().T).amax(-1, keepdim=True) / math.sqrt(D)
    if causal:
      s = s.masked_fill(torch.arange(m, device=DEV)[None] > some[:, None] + (m - n), -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    want, a = p @ vh, p @ vh.abs()
    tol = 2 * (u + (D + 8) * 2.0 ** -23 * size + m * 2.0 ** -24) * a + u * want.abs() + 1e-30
    assert ((out[some, h].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("causal", [False, True])
def test_widest_tiles_over_caches_with_free_rows(causal):
  """Tiles of 256 rows: lengths in use, fewer keys than queries, NaN in every free row of queries and caches."""
  room, used, cache, filled = [2500, 1700], [2300, 1650], [2700, 1800], [2650, 900]
  q, k, v = make(room, cache, 32, 8, 128, torch.bfloat16, 21)
  # (k and v have as many rows as the caches)
  for b in range(2):
    q[sum(room[:b]) + used[b]:sum(room[:b + 1])] = math.nan
    for t in (k, v):
      t[sum(cache[:b]) + filled[b]:sum(cache[:b + 1])] = math.nan
  i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
  out = torch.full_like(q, 7.0)
  ops.packed_attention(q, k, v, offsets(room), offsets(cache), len_q=i32(used), len_k=i32(filled), causal=causal, out=out)
  for b in range(2):
    aq, ak = sum(room[:b]), sum(cache[:b])
    assert (out[aq + used[b]:sum(room[:b + 1])] == 7.0).all()
    sampled(out[aq:aq + used[b]], q[aq:aq + used[b]], k[ak:ak + filled[b]], v[ak:ak + filled[b]], causal)


def test_one_long_sequence_among_empty_ones():
  """Shared key slices of 512 row tiles over 5 million keys: more units of keys than 32-bit floats count one by one."""
  n, m, B = 16384, 5_000_000, 256
  g = torch.Generator(device=DEV).manual_seed(5)
  q, k, v = (torch.randn(t, 1, 8, generator=g, device=DEV, dtype=torch.bfloat16) for t in (n, m, m))
  lens_q, lens_k = [0] * 100 + [n] + [0] * (B - 101), [0] * 100 + [m] + [0] * (B - 101)
  out = ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k))
  for r in torch.arange(0, n, 2000).tolist() + [n - 1]:
    s = q[r, 0].double() @ k[:, 0].double().T / math.sqrt(8)
    p = torch.softmax(s, -1)
    want, a = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
    # (fp32 sums of m terms, whose roundings are of random sign, are split over 4 x slices waves: 2^-24 m / 64 is far above them)
    assert ((out[r, 0].double() - want).abs() <= 2 * (2.0 ** -8 + 2.0 ** -18 + m / 64 * 2.0 ** -24) * a + 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("causal", [False, True])
def test_a_prompt_beside_single_tokens(causal):
  """A piece of a prompt, tokens over long caches, an empty sequence: one call, each as by itself."""
  lens_q, lens_k = [512, 1, 1, 0, 1, 300], [700, 9000, 1, 5, 65, 300]
  q, k, v = make(lens_q, lens_k, 8, 2, 128, torch.bfloat16, 22)
  check(ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal), q, k, v, lens_q, lens_k, causal)
