"""More refusals of the packed-sequence calls: tangents, grids.  Host tensors; nothing here launches a kernel."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from sparsefold_amd import _lib
from sparsefold_amd.backends.hip import ops

BF = torch.bfloat16


class _Launched(Exception):
  pass


@pytest.fixture
def host_tensors(monkeypatch):
  """Argument checks run on host tensors; reaching the library ends the call."""
  def refuse():
    raise _Launched
  monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("cpu"))
  monkeypatch.setattr(ops._lib, "load", refuse)


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(host_tensors, which, no_grad):
  """A dual tensor's tangent would be dropped without a word."""
  q, k, w = torch.ones(6, 4, 32, dtype=BF), torch.ones(6, 4, 32, dtype=BF), torch.ones(32)
  f, pos, cu = ops.rotary_frequencies(32), torch.arange(6), torch.tensor([0, 6], dtype=torch.int32)
  calls = [lambda d, t: ops.packed_attention(d, t, t, cu), lambda d, t: ops.packed_attention(t, t, d, cu),
           lambda d, t: ops.rotary(d, t, pos, f), lambda d, t: ops.rotary(t, d, pos, f),
           lambda d, t: ops.qk_norm_rotary(d, t, w, w, pos, f),
           lambda d, t: ops.qk_norm_rotary(t, t, forward_ad.make_dual(w, w), w, pos, f)]
  with torch.set_grad_enabled(not no_grad):
    with forward_ad.dual_level():
      with pytest.raises(ValueError, match="forward-mode"):
        calls[which](forward_ad.make_dual(q, torch.ones_like(q)), k)
      with pytest.raises(_Launched):                 # inside a dual level, no tangent
        calls[which % 5](q, k)
    with pytest.raises(_Launched):
      calls[which % 5](q, k)


def test_c_attention_refuses_more_workgroups_than_a_grid_holds():
  lib = _lib.load()
  cu = torch.zeros(2, dtype=torch.int32)
  a = _lib.PackedAttentionArgs(B=(1 << 26) // 4 + 1, H=8, Hkv=4, D=8, Tq=1 << 28, Tk=1 << 28, scale=1.0, q=4096, k=4096, v=4096, out=4096,
                               cu_q=cu.data_ptr(), cu_k=cu.data_ptr())
  for s in (a.q_s, a.k_s, a.v_s, a.o_s):
    s[0], s[1] = 64, 8
  assert lib.sf_hip_packed_attention_workspace_bytes(C.byref(a)) == 0
  assert lib.sf_hip_packed_attention_fwd(C.byref(a), None, 0, None) != 0
  buf = C.create_string_buffer(1024)
  lib.sf_hip_last_error(buf, 1024)
  assert "too large for the grid" in buf.value.decode()
