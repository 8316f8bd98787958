"""The residual's addition with the root-mean-square norm against its definition in 64 bits.

The sum is one fp32 addition rounded to the type: equal to the definition's.  The norm is formed in 64 bits and rounded by
way of 32: u = finfo.eps / 2 of the result and 2^-24 more; fp16 results below 2^-14, and 32-bit ones below 2^-126, to half of
the smallest number.  Codes of 8 and 4 bits are equal."""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops
from test_gpu_mx import TYPES, encode, unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda"


def definition(x, r, w, eps):
  h = x.cpu() if r is None else (x.cpu().float() + r.cpu().float()).to(x.dtype)
  d = h.double()
  y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
  return h, y if w is None else y * w.cpu().double()


def near(y, want):
  t = torch.finfo(y.dtype)
  tol = (t.eps / 2 + 2.0 ** -24) * want.abs() + t.smallest_normal * t.eps / 2
  assert ((y.cpu().double() - want).abs() <= tol).all()


def make(shape, dtype, seed=0, size=4.0):
  g = torch.Generator().manual_seed(seed)
  r = lambda k: (k * torch.randn(*shape, generator=g)).to(TYPES[dtype]).to(DEV)
  return r(1.0), r(size), (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(DEV)


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 96), (1, 4096), (8, 4096), (300, 512), (17, 520), (2, 3, 1000), (9, 1024), (7, 2048), (5, 2056), (4, 8192), (3, 8200),
          (3, 16384), (2, 16392), (2, 20001), (1, 70000), (0, 64), (5000, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm(shape, dtype):
  x, r, w = make(shape, dtype, shape[-1])
  for res in (r, None):
    for weight in (w, None):
      y, h = ops.add_rms_norm(x, res, weight, eps=1e-5)
      total, want = definition(x, res, weight, 1e-5)
      near(y, want)
      assert y.shape == x.shape and y.dtype is x.dtype
      assert h is None if res is None else torch.equal(h.cpu(), total)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("output", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (2, 5, 160), (8, 4096), (40, 512), (9, 544), (7, 1024), (6, 2080), (4, 8192), (3, 8224), (3, 16384),
                                   (2, 16416), (1, 65536), (0, 64), (3000, 128)], ids=str)
def test_microscaled(shape, output, dtype):
  x, r, w = make(shape, dtype, shape[-1])
  for res in (r, None):
    for weight in (w, None):
      mx, h = ops.add_rms_norm(x, res, weight, output=output)
      total, want = definition(x, res, weight, 1e-6)
      code, scale = encode(want, output)
      assert torch.equal(mx.scales.cpu().view(torch.uint8), scale) and torch.equal(unpacked(mx), code)
      assert h is None if res is None else torch.equal(h.cpu(), total)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("C", [40, 4096, 20000])
@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -70, 2.0 ** 70, 2.0 ** 120])
def test_rows_whose_squares_leave_32_bits(size, C, dtype):
  g = torch.Generator().manual_seed(C)
  x = (size * torch.randn(4, C, generator=g)).to(TYPES[dtype]).to(DEV)
  y, _ = ops.add_rms_norm(x, None, None, eps=0.0)
  near(y, definition(x, None, None, 0.0)[1])


@pytest.mark.parametrize("C", [64, 4096, 33, 20000])
def test_rows_that_are_not_finite_or_zero(C):
  x = torch.randn(5, C, device=DEV).bfloat16()
  x[1, 3], x[2, 0], x[3] = math.nan, math.inf, 0
  y, _ = ops.add_rms_norm(x, None, None)
  assert torch.isnan(y[1]).all() and torch.isnan(y[2, 0]) and (y[2, 1:] == 0).all() and (y[3] == 0).all()
  assert torch.isfinite(y[0]).all() and torch.isfinite(y[4]).all()
  y, _ = ops.add_rms_norm(x, None, None, eps=0.0)
  assert torch.isnan(y[3]).all()
  if C % 32 == 0:
    mx, _ = ops.add_rms_norm(x, None, None, output="mxfp8")
    s = mx.scales.view(torch.uint8)
    assert (s[1] == 255).all() and s[2, 0] == 255 and (s[2, 1:] == 0).all() and (s[3] == 0).all() and (s[0] != 255).all()


@pytest.mark.parametrize("shape", [(6, 512), (300, 4096), (5, 77), (4, 20000), (2, 3, 64)], ids=str)
def test_in_place_and_given_outputs(shape):
  x, r, w = make(shape, "bf16", 1)
  want_y, want_h = ops.add_rms_norm(x, r, w)
  r2 = r.clone()
  y, h = ops.add_rms_norm(x, r2, w, out_sum=r2)
  assert h is r2 and torch.equal(h, want_h) and torch.equal(y, want_y)
  x2, r2 = x.clone(), r.clone()
  y, h = ops.add_rms_norm(x2, r2, w, out=x2, out_sum=r2)
  assert y is x2 and torch.equal(x2, want_y) and torch.equal(r2, want_h)
  x2, r2 = x.clone(), r.clone()
  y, h = ops.add_rms_norm(x2, r2, w, out=r2, out_sum=x2)
  assert torch.equal(r2, want_y) and torch.equal(x2, want_h)
  x2 = x.clone()
  assert torch.equal(ops.add_rms_norm(x2, r, w, out=x2)[0], want_y)
  if shape[-1] % 32 == 0:
    r2 = r.clone()
    want, _ = ops.add_rms_norm(x, r, w, output="mxfp4")
    mx, h = ops.add_rms_norm(x, r2, w, output="mxfp4", out_sum=r2)
    assert torch.equal(mx.codes, want.codes) and torch.equal(r2, want_h)


@pytest.mark.parametrize("C", [64, 96, 50])
def test_strides_and_alignments(C):
  wide = torch.randn(30, 4, 128, device=DEV).bfloat16()
  w = torch.rand(2 * C, device=DEV)[::2]
  for x, r in ((wide[:, 1, :C], wide[:, 2, :C]), (wide[:, 0, 3:3 + C], wide[:, 3, 8:8 + C]), (wide[::2, 1, 1:1 + C], wide[1::2, 1, :C]),
               (wide.transpose(0, 1)[..., :C], wide.transpose(0, 1)[..., 9:9 + C]), (wide.permute(2, 1, 0)[:C].transpose(0, 2), wide.permute(2, 1, 0)[1:1 + C].transpose(0, 2))):
    y, h = ops.add_rms_norm(x, r, w)
    total, want = definition(x, r, w, 1e-6)
    near(y, want)
    assert torch.equal(h.cpu(), total)
    if C % 32 == 0:
      mx, _ = ops.add_rms_norm(x, r, w, output="mxfp8")
      assert torch.equal(unpacked(mx), encode(want, "mxfp8")[0])
  room = torch.zeros(30, 200, dtype=torch.bfloat16, device=DEV)
  y, _ = ops.add_rms_norm(wide[:, 1, :C], wide[:, 2, :C], w.contiguous(), out=room[:, 7:7 + C])
  assert torch.equal(y, ops.add_rms_norm(wide[:, 1, :C], wide[:, 2, :C], w)[0]) and (room[:, :7] == 0).all() and (room[:, 7 + C:] == 0).all()


def test_capture_and_replay():
  x, r, w = make((64, 4096), "bf16", 2)
  ops.add_rms_norm(x, r, w)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      y, h = ops.add_rms_norm(x, r, w)
      mx, _ = ops.add_rms_norm(y, h, w, output="mxfp8")
  for _ in range(3):
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    y2, h2 = ops.add_rms_norm(x, r, w)
    m2, _ = ops.add_rms_norm(y2, h2, w, output="mxfp8")
    assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(mx.codes.view(torch.uint8), m2.codes.view(torch.uint8))
