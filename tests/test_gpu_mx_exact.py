"""The product of microscaled operands where every sum is exact: equal to the definition's, bit for bit.

Codes are -1, 0 and 1, scales 1/2, 1 and 2 of one operand and 1 of the other, so every product is a multiple of 1/2 up to 2: nothing lies
below 2^-13 of the largest of eight, every partial sum is a multiple of 1/2 below 2^23 and exact in 32 bits whatever the order.  Results stay
below 1024 (asserted), where fp16 holds every multiple of 1/2 (11 bits).  One product lost, counted twice or scaled by another block's
scale changes a result."""
import pytest
import torch

from sparsefold_amd.backends.hip import ops
from test_gpu_mx import DEV, FORMATS

pytestmark = pytest.mark.gpu


def operand(rows, K, format, scaled, g):
  v = torch.randint(-1, 2, (rows, K), generator=g, dtype=torch.int8)
  s = torch.randint(126, 129, (rows, K // 32), generator=g).to(torch.uint8) if scaled else torch.full((rows, K // 32), 127, dtype=torch.uint8)
  if format == "mxfp8":                                        # 1.0 is 0x38
    codes = torch.where(v == 0, 0, torch.where(v > 0, 0x38, 0xB8)).to(torch.uint8).view(torch.float8_e4m3fn)
  else:                                                        # 1.0 is 2
    c = torch.where(v == 0, 0, torch.where(v > 0, 2, 10)).to(torch.uint8)
    codes = c[:, ::2] | (c[:, 1::2] << 4)
  values = v.float() * torch.exp2(s.float() - 127).repeat_interleave(32, dim=1)
  return ops.Microscaled(codes.to(DEV), s.to(DEV)), values


# streamed, up to 16, 32 and 64 rows, 16 and 32 rows of w a workgroup; tiles of 128, whole steps and not, k in parts and not; tiles of 256, one a workgroup and more
SHAPES = [(1, 16, 512), (8, 6200, 1184), (30, 300, 96), (60, 257, 2048), (5, 4097, 544), (16, 4096, 1056), (17, 4113, 672), (30, 5000, 1184), (33, 4099, 512), (64, 7000, 96), (65, 128, 128), (200, 1000, 1600), (100, 520, 4096), (777, 264, 2080), (1000, 700, 640),
          (4230, 4200, 160), (2305, 4104, 1152), (4099, 4104, 640), (4099, 4104, 512), (2570, 4352, 768), (9000, 1032, 512)]


@pytest.mark.parametrize("scaled", ["x", "w"])
@pytest.mark.parametrize("formats", FORMATS, ids="-".join)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_exact_sums(M, N, K, formats, scaled):
  g = torch.Generator().manual_seed(M + K)
  x, a = operand(M, K, formats[0], scaled == "x", g)
  w, b = operand(N, K, formats[1], scaled == "w", g)
  want = a.to(DEV) @ b.to(DEV).t()                             # (as exact: the same multiples of 1/2)
  assert want.abs().max() + 64 < 1024
  y = ops.mx_linear(x, w, dtype=torch.float16)
  assert torch.equal(y.float(), want)
  bias = torch.randint(-64, 64, (N,), generator=g).float().to(DEV)
  y = ops.mx_linear(x, w, bias, dtype=torch.float16)
  assert torch.equal(y.float(), want + bias)
