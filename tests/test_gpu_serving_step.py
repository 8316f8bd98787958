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


# ---- the calls' common form in the host module against ctypes ------------------------------------------

def forms(name):
  """Arguments that the host module takes."""
  g = torch.Generator().manual_seed(5)
  r = lambda *s, dtype=BF: torch.randn(*s, generator=g).to(dtype).to(DEV)
  if name == "norm":
    for shape, dtype in (((8, 512), BF), ((3, 5, 96), torch.float16), ((64,), torch.float32), ((2, 77), BF)):
      x = r(*shape, dtype=dtype)
      for residual in (r(*shape, dtype=dtype), None):
        for weight in (r(shape[-1], dtype=torch.float32), None):
          for output in (None,) if shape[-1] % 32 else (None, "mxfp8", "mxfp4"):
            yield (x, residual, weight, 1e-5, output), lambda: ops.add_rms_norm(x, residual, weight, eps=1e-5, output=output)
  elif name == "quantize":
    for shape, dtype in (((7, 64), BF), ((2, 3, 128), torch.float32), ((32,), torch.float16)):
      x = r(*shape, dtype=dtype)
      for f in ("mxfp8", "mxfp4"):
        yield (x, f), lambda: ops.mx_quantize(x, f)
  elif name == "dequantize":
    for shape in ((7, 64), (2, 3, 128), (32,)):
      for f in ("mxfp8", "mxfp4"):
        x = ops.mx_quantize(r(*shape), f)
        for dtype in (BF, torch.float16, torch.float32):
          yield (*x, dtype), lambda: ops.mx_dequantize(x, dtype)
  elif name == "linear":
    for lead, N, K in (((8,), 100, 256), ((2, 100), 256, 4096), ((), 64, 64), ((300,), 64, 1024)):
      for fx, fw in mx.FORMATS:
        x, w = ops.mx_quantize(r(*lead, K), fx), ops.mx_quantize(r(N, K), fw)
        for bias in (r(N, dtype=torch.float32), None):
          for dtype in (BF, torch.float16):
            yield (*x, *w, bias, dtype), lambda: ops.mx_linear(x, w, bias, dtype=dtype)
  else:
    for T, lens, heads, layout in ((4, [1, 1, 1, 1], 4, "rows"), (90, [70, 1, 0, 19], 2, "both"), (1, [1, 0, 0, 0], 1, "heads")):
      shape = {"rows": (40, 16, heads, 64), "both": (40, 2, 16, heads, 64), "heads": (40, heads, 16, 64)}[layout]
      kp, vp = r(*shape), r(*shape)
      kp, vp = (kp[:, 0], kp[:, 1]) if layout == "both" else (kp.transpose(1, 2), vp.transpose(1, 2)) if layout == "heads" else (kp, vp)
      table = torch.randperm(40, generator=g)[:32].view(4, 8).to(torch.int32).to(DEV)
      cu, len_k = attention.offsets(lens), ints([100, 30, 128, 19])
      y = r(T, 6 * heads, 64)
      q, k, v = y[:, :4 * heads], y[:, 4 * heads:5 * heads], y[:, 5 * heads:]
      if name == "write":
        for new in (None, ints([1, 1, 0, 3])):
          def write():
            a, b = kp.clone(), vp.clone()
            ops.paged_cache_write(k, v, kp, vp, table, cu, len_k, len_new=new)
            result = kp.clone(), vp.clone()
            kp.copy_(a)
            vp.copy_(b)
            return result
          yield (k, v, kp, vp, table, cu, len_k, new), write
      else:
        for len_q, causal, scale, most in ((None, True, None, None), (ints([1, 1, 0, 3]), False, 0.25, 128), (None, True, None, 0)):
          def call():                                          # (rows outside every sequence hold what was there)
            out = ops.paged_attention(q, kp, vp, table, cu, len_k, len_q=len_q, causal=causal, scale=scale, max_len=most)
            rows = [i for b, n in enumerate(lens) for i in range(int(cu[b]), int(cu[b]) + (n if len_q is None else min(n, int(len_q[b]))))]
            return out[rows]
          yield (q, kp, vp, table, cu, len_k, len_q, causal, scale, most), call


CALLS = {"norm": "add_rms_norm", "quantize": "mx_quantize", "dequantize": "mx_dequantize", "linear": "mx_linear", "write": "paged_cache_write", "attention": "paged_attention"}


def flat(x):
  return [t for y in x for t in flat(y)] if isinstance(x, tuple) else [] if x is None else [x]


@pytest.mark.parametrize("name", list(CALLS))
def test_host_module_gives_what_ctypes_gives(name, monkeypatch):
  ops._library()
  assert ops._front
  for args, call in forms(name):
    assert getattr(ops._front, CALLS[name])(*args) is not None
    got = call()
    with monkeypatch.context() as m:
      m.setattr(ops, "_front", False)
      want = call()
    for a, b in zip(flat(got), flat(want), strict=True):
      assert a.shape == b.shape and a.dtype is b.dtype and a.is_contiguous() and torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)
    assert type(got) is type(want)


def test_host_module_leaves_other_forms():
  """Copies, gradients, other devices' and wrong tensors are the wrapper's."""
  ops._library()
  x, w = torch.randn(4, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV)
  norm_of = ops._front.add_rms_norm
  for args in ((x.t()[:4].contiguous().t(), None, None, 1e-6, None), (x[:, ::2], None, None, 1e-6, None), (x, x[:2], None, 1e-6, None), (x, x.half(), None, 1e-6, None),
               (x, None, w[:32], 1e-6, None), (x, None, w.double(), 1e-6, None), (x, None, w, -1.0, None), (x, None, w, math.nan, None), (x, None, w, 1, None),
               (x, None, w, 1e-6, "mxfp6"), (x, None, w, 1e-6, True), (x.cpu(), None, None, 1e-6, None), (x, x.cpu(), None, 1e-6, None), (x, None, None, 1e-6), ("x", None, w, 1e-6, None),
               (x[:0], None, None, 1e-6, None), (x.clone().requires_grad_(), None, None, 1e-6, None), (x, None, w.clone().requires_grad_(), 1e-6, None),
               (x[1:].view(-1)[4:36 + 96].view(2, 64), None, None, 1e-6, "mxfp8")):
    assert norm_of(*args) is None
  with pytest.raises(ValueError, match="no backward pass"):
    ops.add_rms_norm(x.clone().requires_grad_(), None, None)
  with torch.no_grad():
    assert norm_of(x.clone().requires_grad_(), None, None, 1e-6, None) is not None
  import torch.autograd.forward_ad as fwd
  with fwd.dual_level():
    assert norm_of(fwd.make_dual(torch.ones(2, 32, device=DEV), torch.ones(2, 32, device=DEV)), None, None, 1e-6, None) is None
  with torch.inference_mode():
    y, _ = ops.add_rms_norm(x, None, w)
    assert y.is_inference()


def test_writes_are_seen_by_autograd():
  """Pages that a graph saved are not used behind a write, by either way."""
  ops._library()
  k = torch.randn(1, 2, 64, device=DEV, dtype=BF)
  pages = [torch.zeros(2, 16, 2, 64, device=DEV, dtype=BF) for _ in range(2)]
  before = [t._version for t in pages]
  ops.paged_cache_write(k, k, *pages, ints([[0]]), ints([0, 1]), ints([1]))
  assert all(t._version > n for t, n in zip(pages, before))
  s = torch.ones((), device=DEV, requires_grad=True)
  loss = (pages[0].float() * s).sum() + (pages[0] * s.to(BF)).sum()
  ops.paged_cache_write(k, k, *pages, ints([[0]]), ints([0, 1]), ints([1]))
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    loss.backward()


def test_streams_of_the_host_module():
  """A call runs on the stream that is current where it is made."""
  ops._library()
  side = torch.cuda.Stream()
  x = torch.randn(4096, 4096, device=DEV).to(BF)
  want = ops.mx_quantize(x.clone().mul_(2), "mxfp8")
  torch.cuda.synchronize()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(20):
      x.mul_(1.0)
    x.mul_(2)
    got = ops.mx_quantize(x, "mxfp8")
  side.synchronize()
  assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scales.view(torch.uint8), want.scales.view(torch.uint8))
