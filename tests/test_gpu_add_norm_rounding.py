"""The norm's results in 16 bits are those of one rounding of its 64-bit value.

Both sides form the norm in 64 bits, within some 2^-51 of each other, and round it to the nearest number, ties to even: a result
can differ only where the value lies that close to a border, which in 2^21 results happens in one of 2^18 runs at most with the 8
or 11 bits that are kept.  By way of 32 bits, 1 of 2^17 (bf16) or 2^14 (fp16) results goes to the wrong side."""
import pytest
import torch

from sparsefold_amd.backends.hip import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BITS = {torch.bfloat16: (8, -126), torch.float16: (11, -14)}   # of a number, exponent of the smallest normal one


def rounded(y, dtype):
  """64 bits to the nearest number of the type at once (none of the values overflows)."""
  bits, least = BITS[dtype]
  e = torch.frexp(y)[1].clamp(min=least + 1) - bits
  return torch.ldexp(torch.ldexp(y, -e.double()).round(), e.double()).to(dtype)


@pytest.mark.parametrize("dtype", list(BITS), ids=str)
@pytest.mark.parametrize("rows,C", [(32768, 64), (4096, 520), (1024, 2048), (256, 8192), (128, 16384), (512, 4095), (99, 20001), (3000, 700)])
def test_one_rounding(rows, C, dtype):
  g = torch.Generator().manual_seed(C)
  x, r = (torch.randn(rows, C, generator=g).to(dtype) for _ in range(2))
  w = 1 + 0.3 * torch.randn(C, generator=g)
  for residual, weight in ((r, w), (None, w), (r, None)):
    y, h = ops.add_rms_norm(x.to(DEV), None if residual is None else residual.to(DEV), None if weight is None else weight.to(DEV), eps=2.0 ** -20)
    d = (x if h is None else h.cpu()).double()
    want = d / torch.sqrt(d.square().mean(-1, keepdim=True) + 2.0 ** -20)
    if weight is not None:
      want = want * weight.double()
      assert not torch.equal(rounded(want, dtype), want.float().to(dtype))        # (the inputs have results that two roundings change)
    assert torch.equal(y.cpu(), rounded(want, dtype))


def test_tiny_results_in_one_rounding():
  """Results among fp16's subnormal numbers and around its smallest normal one."""
  g = torch.Generator().manual_seed(1)
  x = torch.randn(2048, 1024, generator=g).half()
  w = torch.exp2(-14 - 12 * torch.rand(1024, generator=g))
  y, _ = ops.add_rms_norm(x.to(DEV), None, w.to(DEV), eps=0.0)
  d = x.double()
  want = d / torch.sqrt(d.square().mean(-1, keepdim=True)) * w.double()
  assert not torch.equal(rounded(want, torch.float16), want.float().half())
  assert torch.equal(y.cpu(), rounded(want, torch.float16))
