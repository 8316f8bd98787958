"""The calls of a serving step together, as a decoder layer runs them: residual with the norm, projections of microscaled
numbers, norm of the heads with their rotary positions, the paged cache and its attention.  Each call's result is checked
against its definition in 64 bits from what the call before it gave, with the tolerances of its own tests."""
import math

import pytest
import torch

import test_gpu_add_norm as norm
import test_gpu_mx as mx
import test_gpu_packed_attention as attention
import test_gpu_rotary as rotary
from sparsefold_amd.backends.hip import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


class Layer:
  """A layer's weights and its cache; ``step`` runs the tokens of a batch through it."""

  def __init__(self, C, H, Hk, D, page, sequences, cols, x_format, w_format):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)
    weight = lambda n, k: ops.mx_quantize(r(n, k) * k ** -0.5, w_format)
    self.C, self.H, self.Hk, self.D, self.format = C, H, Hk, D, x_format
    self.qkv, self.o, self.up, self.down = weight((H + 2 * Hk) * D, C), weight(C, H * D), weight(2 * C, C), weight(C, 2 * C)
    self.bias = 0.1 * r((H + 2 * Hk) * D)
    self.n1, self.n2, self.nq, self.nk = (1 + 0.1 * r(n) for n in (C, C, D, D))
    self.freqs = ops.rotary_frequencies(D, device=DEV)
    pages = sequences * cols + 2
    self.k, self.v = (torch.full((pages, page, Hk, D), math.nan, dtype=BF, device=DEV) for _ in range(2))
    self.table = torch.randperm(pages, generator=g)[:sequences * cols].view(sequences, cols).to(torch.int32).to(DEV)

  def step(self, x, residual, cu, len_k, positions, len_new=None, seen=lambda *a: None):
    H, Hk, D = self.H, self.Hk, self.D
    a, h = ops.add_rms_norm(x, residual, self.n1, output=self.format)
    seen("norm", x, residual, self.n1, a, h)
    y = ops.mx_linear(a, self.qkv, self.bias)
    seen("linear", a, self.qkv, self.bias, y)
    y = y.view(-1, H + 2 * Hk, D)
    before = y.clone()
    q, k = ops.qk_norm_rotary(y[:, :H], y[:, H:H + Hk], self.nq, self.nk, positions, self.freqs, out_q=y[:, :H], out_k=y[:, H:H + Hk])
    seen("rotary", before[:, :H], self.nq, q, positions)
    seen("rotary", before[:, H:H + Hk], self.nk, k, positions)
    ops.paged_cache_write(k, y[:, H + Hk:], self.k, self.v, self.table, cu, len_k, len_new=len_new)
    out = torch.zeros_like(y[:, :H], memory_format=torch.contiguous_format)   # (rows behind a padded sequence's tokens stay)
    ops.paged_attention(q, self.k, self.v, self.table, cu, len_k, len_q=len_new, out=out)
    seen("attention", q, k, y[:, H + Hk:], out)
    a = ops.mx_quantize(out.view(-1, H * D), self.format)
    seen("quantize", out.view(-1, H * D), a)
    y = ops.mx_linear(a, self.o)
    seen("linear", a, self.o, None, y)
    a, h = ops.add_rms_norm(y, h, self.n2, output=self.format, out_sum=h)
    u = torch.nn.functional.silu(ops.mx_linear(a, self.up))
    a = ops.mx_quantize(u, self.format)
    y = ops.mx_linear(a, self.down)
    seen("linear", a, self.down, None, y)
    return y, h


def ints(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("formats", mx.FORMATS, ids="-".join)
@pytest.mark.parametrize("page", [16, 48])
def test_prompts_pieces_and_tokens(page, formats):
  """Prompts of odd lengths, single tokens, a further piece beside tokens, and a padded batch, over one cache."""
  layer = Layer(256, 4, 2, 64, page, 4, 20, *formats)
  g = torch.Generator().manual_seed(1)
  cache = [[torch.zeros(0, 2, 64, dtype=BF)] * 2 for _ in range(4)]
  for lens, padded in (([37, 5, 1, 130], None), ([1, 1, 1, 1], None), ([1, 1, 70, 0], None), ([1, 2, 0, 1], 3), ([1, 1, 1, 1], None)):
    starts = [padded * b for b in range(5)] if padded else [sum(lens[:b]) for b in range(5)]
    T = starts[-1]
    x, residual = (torch.randn(T, 256, generator=g).to(BF).to(DEV) for _ in range(2))
    past = [c[0].shape[0] for c in cache]
    positions = torch.zeros(T, dtype=torch.int32)
    for b, n in enumerate(lens):
      positions[starts[b]:starts[b] + n] = torch.arange(past[b], past[b] + n)
    count = []

    def seen(kind, *a):
      count.append(kind)
      if kind == "norm":
        total, want = norm.definition(*a[:3], 1e-6)
        assert torch.equal(a[4].cpu(), total)
        mx.same(a[3], want)
      elif kind == "linear":
        mx.check(a[3], a[0], a[1], a[2])
      elif kind == "rotary":
        rotary.check(a[2], a[0], a[3], layer.freqs, norm="rms", weight=a[1])
      elif kind == "quantize":
        mx.same(a[1], a[0])
      else:
        q, k, v, out = a
        for b, n in enumerate(lens):
          rows = slice(starts[b], starts[b] + n)
          cache[b] = [torch.cat((old, new[rows].cpu())) for old, new in zip(cache[b], (k, v))]
          want, tol = attention.definition(q[rows], *cache[b], True, 1 / 8)
          assert ((out[rows].cpu().double() - want).abs() <= tol).all(), f"sequence {b}"
          assert (out[starts[b] + n:starts[b + 1]] == 0).all()

    y, h = layer.step(x, residual, ints(starts), ints([p + n for p, n in zip(past, lens)]), positions.to(DEV), ints(lens) if padded else None, seen)
    assert len(count) == 8 and torch.isfinite(y).all() and torch.isfinite(h).all()


@pytest.mark.parametrize("formats", mx.FORMATS, ids="-".join)
def test_captured_step(formats):
  """A captured step, replayed with other tokens, lengths and pages, gives what the calls give one by one."""
  layer, eager = (Layer(512, 8, 2, 64, 16, 3, 30, *formats) for _ in range(2))
  for one in (layer, eager):
    one.k.zero_()
    one.v.zero_()
  cu, len_k, positions = ints([0, 1, 2, 3]), ints([1, 1, 1]), ints([0, 0, 0])
  x, residual = (torch.zeros(3, 512, dtype=BF, device=DEV) for _ in range(2))
  layer.step(x, residual, cu, len_k, positions)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = layer.step(x, residual, cu, len_k, positions)
  layer.k.zero_()
  layer.v.zero_()
  g = torch.Generator().manual_seed(2)
  lens = [0, 200, 17]
  for i in range(6):
    lens = [n + 1 for n in lens]
    x.copy_(torch.randn(3, 512, generator=g))
    residual.copy_(torch.randn(3, 512, generator=g))
    len_k.copy_(ints(lens))
    positions.copy_(ints([n - 1 for n in lens]))
    graph.replay()
    torch.cuda.synchronize()
    want = eager.step(x, residual, cu, len_k, positions)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert torch.equal(layer.k, eager.k) and torch.equal(layer.v, eager.v)
    assert torch.isfinite(out[0]).all()
