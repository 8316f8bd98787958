"""Sizes that the serving-step calls refuse by name; nothing here launches a kernel or holds the tensors' memory."""
import pytest
import torch

from sparsefold_amd.backends.hip import ops

U8 = torch.uint8


@pytest.fixture(autouse=True)
def meta_tensors(monkeypatch):
  def refuse():
    raise AssertionError("reached the library")
  monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("meta"))
  monkeypatch.setattr(ops._lib, "load", refuse)
  monkeypatch.setattr(ops, "_front", False)


@pytest.mark.parametrize("format", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("K", [1 << 31, (1 << 32) + 32])
def test_rows_longer_than_the_kernels_count(K, format):
  with pytest.raises(ValueError, match="2\\^31"):
    ops.mx_quantize(torch.empty(1, K, dtype=torch.bfloat16, device="meta"), format)
  codes = torch.empty(1, K, device="meta", dtype=torch.float8_e4m3fn) if format == "mxfp8" else torch.empty(1, K // 2, device="meta", dtype=U8)
  with pytest.raises(ValueError, match="2\\^31"):
    ops.mx_dequantize(ops.Microscaled(codes, torch.empty(1, K // 32, device="meta", dtype=U8)))
