"""Rotary positions and the norm before them at the ends of sizes and of the number range; tolerance of
test_gpu_rotary."""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops
from tests.test_gpu_rotary import DEV, TYPES, check, rand

pytestmark = pytest.mark.gpu


def test_more_workgroups_than_a_launch_dimension_holds():
  """2^26 tokens: 2^24 workgroups of 256 threads and one.  The first, those on both sides of each grid row's border, the last."""
  T, D = (1 << 26) + 3, 8
  q = torch.randn(T, 1, D, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV, dtype=torch.bfloat16)
  pos, f = torch.arange(T, dtype=torch.int32, device=DEV), ops.rotary_frequencies(D, device=DEV)
  oq, _ = ops.rotary(q, None, pos, f)
  for start in (0, (1 << 24) - 500, (1 << 25) - 500, 3 * (1 << 24) - 500, T - 1000):
    s = slice(start, start + 1000)
    check(oq[s], q[s], pos[s], f)


@pytest.mark.parametrize("dtype,size", [("bf16", 2.0 ** 120), ("fp32", 2.0 ** 100), ("bf16", 2.0 ** 66), ("fp32", 2.0 ** -90), ("bf16", 2.0 ** -110)])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dims", [(128, 128), (64, 32), (255, 30)], ids=lambda d: "x".join(map(str, d)))
def test_norm_of_values_whose_squares_leave_the_range(dims, norm, dtype, size):
  """The sum of squares passes fp32, or vanishes: the normed head is of ordinary size.  Ordinary heads beside them."""
  D, R = dims
  q, k = rand(6, 4, D, dtype=TYPES[dtype]), rand(6, 3, D, dtype=TYPES[dtype], seed=1)
  q[:, ::2] *= size
  k[1::2] *= size
  q[4, 1, 3], q[4, 2, 3] = math.inf, math.nan
  pos, f = torch.arange(6, device=DEV), ops.rotary_frequencies(R, device=DEV)
  w, b = 1 + 0.3 * rand(D, seed=2), rand(D, seed=3) if norm == "layer" else None
  eps = 1e-6 if size > 1 else 0.0
  oq, ok = ops.qk_norm_rotary(q, k, w, w, pos, f, norm=norm, eps=eps, q_bias=b, k_bias=b)
  assert not torch.isfinite(oq[4, 1].float()).all() and not torch.isfinite(oq[4, 2].float()).all()
  rows = [0, 1, 2, 3, 5]
  check(oq[rows], q[rows], pos[rows], f, norm=norm, weight=w, bias=b, eps=eps)
  check(ok, k, pos, f, norm=norm, weight=w, bias=b, eps=eps)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("value", [0.0, 2.0 ** 125, -2.0 ** 127, 2.0 ** -120])
def test_norm_of_heads_of_one_value(value, dtype):
  """Layer norm: zero, whatever the value; rms: its sign (its size over eps's root where it is small)."""
  q = torch.full((3, 2, 64), value, dtype=TYPES[dtype], device=DEV)
  pos, f = torch.arange(3, device=DEV), ops.rotary_frequencies(64, device=DEV)
  for norm in ("rms", "layer"):
    oq, _ = ops.qk_norm_rotary(q, None, None, None, pos, f, norm=norm)
    check(oq, q, pos, f, norm=norm)
