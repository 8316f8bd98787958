"""Views whose values are negated when read (imaginary parts of a lazily conjugated tensor) through the serving-step calls."""
import pytest
import torch

from sparsefold_amd.backends.hip import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def imaginary(*shape):
  t = torch.randn(*shape, dtype=torch.complex64, device=DEV).conj().imag
  assert t.is_neg()
  return t


@pytest.mark.parametrize("shape", [(1, 1), (5, 1), (1,), (7, 64)], ids=str)
def test_norm(shape):
  x, r, w = imaginary(*shape), imaginary(*shape), imaginary(shape[-1])
  for args in ((x, r, w), (x, None, w), (x.resolve_neg(), r, None), (x.resolve_neg(), None, w)):
    plain = tuple(t if t is None else t.resolve_neg() for t in args)
    y, h = ops.add_rms_norm(*args)
    want, total = ops.add_rms_norm(*plain)
    assert torch.equal(y, want) and (h is None) == (total is None) and (h is None or torch.equal(h, total))


def test_quantize_and_bias():
  x, w = imaginary(3, 64), torch.randn(1, 64, device=DEV)
  for t in (x, torch._neg_view(x.resolve_neg())):
    for f in ("mxfp8", "mxfp4"):
      a, b = ops.mx_quantize(t, f), ops.mx_quantize(t.resolve_neg(), f)
      assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8))
  x, w, bias = ops.mx_quantize(x, "mxfp8"), ops.mx_quantize(w, "mxfp4"), imaginary(1)
  assert torch.equal(ops.mx_linear(x, w, bias), ops.mx_linear(x, w, bias.resolve_neg()))


def test_outputs_are_refused():
  x = torch.randn(4, 1, device=DEV)
  for kw in (dict(out=imaginary(4, 1)), dict(out_sum=imaginary(4, 1))):
    with pytest.raises(ValueError, match="negated"):
      ops.add_rms_norm(x, x.clone(), None, **kw)
  codes = ops.mx_quantize(torch.randn(4, 32, device=DEV))
  with pytest.raises(ValueError, match="negated"):
    ops.mx_linear(codes, ops.mx_quantize(torch.randn(1, 32, device=DEV)), out=torch._neg_view(torch.zeros(4, 1, dtype=torch.float16, device=DEV)))
