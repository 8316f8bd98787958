"""The host module beside other threads of the interpreter."""
import ctypes as C
import shutil
import threading

import pytest
import torch

from sparsefold_amd import _lib
from sparsefold_amd.backends.hip import ops
from test_gpu_serving_step import BF, CALLS, DEV, flat, forms

pytestmark = pytest.mark.gpu


@pytest.fixture
def lock_reporter(tmp_path, monkeypatch):
  """A copy of the host module, its entries in the place of the library's: each answers whether its thread holds the interpreter's
  lock, which the calls take for a status.  No kernel is launched."""
  lib = ops._library()                                         # (the calls that make arguments keep the module of their own)
  copy = tmp_path / "front_of_the_lock.so"
  shutil.copy(_lib.front_path(), copy)
  monkeypatch.setattr(_lib, "front_path", lambda: copy)
  asked = C.cast(C.pythonapi.PyGILState_Check, C.c_void_p).value
  module = _lib.front(lib, ops.Microscaled)
  module.bind(C.cast(lib.sf_hip_last_error, C.c_void_p).value, *[asked] * (len(_lib._FRONT) - 1), ops.Microscaled)
  return module


@pytest.mark.parametrize("name", list(CALLS))
def test_host_module_runs_without_the_interpreters_lock(name, lock_reporter):
  """Other Python threads go on while a call allocates and launches, as through ctypes."""
  for args, _ in forms(name):
    assert getattr(lock_reporter, CALLS[name])(*args) is not None


def test_host_module_called_by_threads_at_once():
  ops._library()
  x, w = torch.randn(64, 512, device=DEV).to(BF), torch.rand(512, device=DEV)
  want = flat((ops.add_rms_norm(x, x, w, output="mxfp8"), ops.mx_dequantize(ops.mx_quantize(x))))
  torch.cuda.synchronize()
  got = [None] * 4
  def work(i):
    for _ in range(200):
      got[i] = flat((ops.add_rms_norm(x, x, w, output="mxfp8"), ops.mx_dequantize(ops.mx_quantize(x))))
  threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  torch.cuda.synchronize()
  for g in got:
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(g, want, strict=True))
