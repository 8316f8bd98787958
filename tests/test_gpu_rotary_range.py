"""Rotary positions and the norm before them at the ends of sizes and of the number range; tolerance of
test_gpu_rotary."""
import pytest
import torch

from sparsefold_amd.backends.hip import ops
from tests.test_gpu_rotary import DEV, check

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
