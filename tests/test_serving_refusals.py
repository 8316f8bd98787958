"""Refused arguments of the serving-step calls (paged cache, microscaled numbers, residual with the norm), and what their
kernels' index arithmetic assumes; nothing here launches a kernel."""
import ctypes as C
import math

import pytest
import torch

from sparsefold_amd import _lib
from sparsefold_amd.backends.hip import ops

BF, F8, U8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8, torch.int32


class _Launched(Exception):
  pass


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch, request):
  """Argument checks run on host tensors; reaching the library ends the call."""
  if "lib" in request.fixturenames:
    return
  def refuse():
    raise _Launched
  monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("cpu"))
  monkeypatch.setattr(ops._lib, "load", refuse)


def ints(*x):
  return torch.tensor(x, dtype=I32)


def attention_args(**kw):
  a = dict(q=torch.zeros(6, 4, 32, dtype=BF), k_pages=torch.zeros(5, 16, 2, 32, dtype=BF), v_pages=torch.zeros(5, 16, 2, 32, dtype=BF),
           page_table=torch.zeros(2, 3, dtype=I32), cu_q=ints(0, 2, 6), len_k=ints(20, 40))
  a.update(kw)
  return a


def write_args(**kw):
  a = dict(k=torch.zeros(6, 2, 32, dtype=BF), v=torch.zeros(6, 2, 32, dtype=BF), k_pages=torch.zeros(5, 16, 2, 32, dtype=BF),
           v_pages=torch.zeros(5, 16, 2, 32, dtype=BF), page_table=torch.zeros(2, 3, dtype=I32), cu=ints(0, 2, 6), len_k=ints(20, 40))
  a.update(kw)
  return a


def test_device_tensors_are_needed(monkeypatch):
  monkeypatch.undo()
  for call, args in ((ops.paged_attention, attention_args()), (ops.paged_cache_write, write_args())):
    with pytest.raises(ValueError, match="device tensors"):
      call(**args)
  x = torch.zeros(2, 32)
  for call in (lambda: ops.add_rms_norm(x, x, None), lambda: ops.mx_quantize(x), lambda: ops.mx_dequantize(mx(2, 32)), lambda: ops.mx_linear(mx(2, 32), mx(3, 32))):
    with pytest.raises(ValueError, match="device tensors"):
      call()


def test_accepted_arguments_reach_the_library():
  both = torch.zeros(5, 2, 16, 2, 32, dtype=BF)
  heads = torch.zeros(5, 2, 16, 32, dtype=BF)
  for kw in ({}, dict(len_q=ints(1, 2)), dict(out=torch.zeros(6, 8, 32, dtype=BF)[:, ::2]), dict(max_len=7), dict(max_len=0), dict(causal=False, scale=0.5),
             dict(k_pages=both[:, 0], v_pages=both[:, 1]), dict(k_pages=heads.transpose(1, 2), v_pages=heads.transpose(1, 2))):
    with pytest.raises(_Launched):
      ops.paged_attention(**attention_args(**kw))
  fused = torch.zeros(6, 4, 32, dtype=BF)
  for kw in ({}, dict(len_new=ints(1, 2)), dict(k=fused[:, :2], v=fused[:, 2:]), dict(k_pages=both[:, 0], v_pages=both[:, 1])):
    with pytest.raises(_Launched):
      ops.paged_cache_write(**write_args(**kw))
  x = torch.zeros(3, 4, 64, dtype=BF)
  for kw in ({}, dict(output="mxfp8"), dict(output="mxfp4", out_sum=x), dict(out=x), dict(eps=0.0)):
    with pytest.raises(_Launched):
      ops.add_rms_norm(x, torch.zeros_like(x), torch.ones(64), **kw)
  for f in ("mxfp8", "mxfp4"):
    with pytest.raises(_Launched):
      ops.mx_quantize(x, f)
  with pytest.raises(_Launched):
    ops.mx_linear(mx(3, 64), mx(5, 64, False), torch.zeros(5))


CACHE = [
    (dict(k_pages=torch.zeros(5, 16, 64, dtype=BF)), "pages, rows, heads, dim"),
    (dict(v_pages=torch.zeros(4, 16, 2, 32, dtype=BF)), "alike"),
    (dict(v_pages=torch.zeros(5, 16, 2, 32, dtype=torch.float16)), "alike"),
    (dict(k_pages=torch.zeros(5, 8, 2, 32, dtype=BF), v_pages=torch.zeros(5, 8, 2, 32, dtype=BF)), "multiple of 16 rows"),
    (dict(k_pages=torch.zeros(5, 40, 2, 32, dtype=BF), v_pages=torch.zeros(5, 40, 2, 32, dtype=BF)), "multiple of 16 rows"),
    (dict(k_pages=torch.zeros(0, 16, 2, 32, dtype=BF), v_pages=torch.zeros(0, 16, 2, 32, dtype=BF)), "multiple of 16 rows"),
    (dict(k_pages=torch.zeros(5, 16, 2, 36, dtype=BF)[..., :32], v_pages=torch.zeros(5, 16, 2, 36, dtype=BF)[..., :32]), "16-byte aligned"),
    (dict(k_pages=torch.zeros(5, 16, 2, 64, dtype=BF)[..., ::2], v_pages=torch.zeros(5, 16, 2, 64, dtype=BF)[..., ::2]), "16-byte aligned"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), "page_table"),
    (dict(page_table=torch.zeros(3, 3, dtype=I32)), "page_table"),
    (dict(page_table=torch.zeros(2, 0, dtype=I32)), "page_table"),
    (dict(page_table=torch.zeros(1, 1, dtype=I32).expand(2, (1 << 26) + 1)), "2\\^30"),
    (dict(len_k=ints(1, 2, 3)), "len_k"),
    (dict(len_k=torch.zeros(2, dtype=torch.int64)), "len_k"),
]


@pytest.mark.parametrize("kw,match", CACHE + [
    (dict(q=torch.zeros(6, 128, dtype=BF)), "tokens, heads, dim"),
    (dict(q=torch.zeros(6, 4, 32)), "bfloat16 or float16"),
    (dict(q=torch.zeros(6, 3, 32, dtype=BF)), "evenly"),
    (dict(q=torch.zeros(6, 4, 64, dtype=BF)), "one head dim"),
    (dict(cu_q=torch.tensor([0, 2, 6])), "int32"),
    (dict(cu_q=ints(0)), "two offsets"),
    (dict(len_q=ints(1)), "len_q"),
    (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(max_len=-1), "max_len"),
    (dict(out=torch.zeros(6, 4, 32)), "out must be"),
    (dict(out=torch.zeros(5, 4, 32, dtype=BF)), "out must be"),
    (dict(out=torch.zeros(1, 4, 32, dtype=BF).expand(6, 4, 32)), "out must be"),
])
def test_attention_refuses(kw, match):
  with pytest.raises(ValueError, match=match):
    ops.paged_attention(**attention_args(**kw))


@pytest.mark.parametrize("kw,match", CACHE + [
    (dict(k=torch.zeros(6, 64, dtype=BF)), "tokens, heads, dim"),
    (dict(v=torch.zeros(5, 2, 32, dtype=BF)), "tokens, heads, dim"),
    (dict(k=torch.zeros(6, 2, 32), v=torch.zeros(6, 2, 32)), "bfloat16 or float16"),
    (dict(k=torch.zeros(6, 3, 32, dtype=BF), v=torch.zeros(6, 3, 32, dtype=BF)), "against"),
    (dict(k=torch.zeros(6, 2, 16, dtype=BF), v=torch.zeros(6, 2, 16, dtype=BF)), "against"),
    (dict(cu=ints(0)), "two offsets"),
    (dict(len_new=ints(1)), "len_new"),
    (dict(k_pages=torch.zeros(1, 16, 2, 32, dtype=BF).expand(5, 16, 2, 32), v_pages=torch.zeros(5, 16, 2, 32, dtype=BF)), "once"),
])
def test_write_refuses(kw, match):
  with pytest.raises(ValueError, match=match):
    ops.paged_cache_write(**write_args(**kw))


@pytest.mark.parametrize("D", [0, 4, 20, 136, 256])
def test_head_dims_are_refused(D):
  pages = torch.zeros(5, 16, 2, D, dtype=BF)
  with pytest.raises(ValueError, match="head dim|16-byte"):
    ops.paged_attention(**attention_args(q=torch.zeros(6, 4, D, dtype=BF), k_pages=pages, v_pages=pages))


def test_overlaps_are_refused():
  a = attention_args()
  with pytest.raises(ValueError, match="overlaps"):
    ops.paged_attention(**a, out=a["q"])
  with pytest.raises(ValueError, match="overlaps"):
    ops.paged_attention(**a, out=a["k_pages"].view(-1, 4, 32)[:6])
  one = torch.zeros(5, 16, 2, 32, dtype=BF)
  with pytest.raises(ValueError, match="k_pages and v_pages overlap"):
    ops.paged_cache_write(**write_args(k_pages=one, v_pages=one))
  wide = torch.zeros(5, 16, 3, 32, dtype=BF)
  with pytest.raises(ValueError, match="overlap"):
    ops.paged_cache_write(**write_args(k_pages=wide[:, :, :2], v_pages=wide[:, :, 1:]))
  with pytest.raises(ValueError, match="pages overlap k or v"):
    ops.paged_cache_write(**write_args(k_pages=one, k=one.view(-1, 2, 32)[:6]))
  x, r, w = torch.zeros(6, 64, dtype=BF), torch.zeros(6, 64, dtype=BF), torch.ones(64)
  wide = torch.zeros(7, 64, dtype=BF)
  for kw in (dict(out=x, out_sum=x), dict(out=wide[:6], out_sum=wide[1:])):
    with pytest.raises(ValueError, match="overlap"):
      ops.add_rms_norm(x, r, w, **kw)
  with pytest.raises(ValueError, match="overlap nothing else"):
    ops.add_rms_norm(wide[:6], r, w, out=wide[1:])
  f = torch.zeros(6, 64)
  with pytest.raises(ValueError, match="weight"):
    ops.add_rms_norm(f, f.clone(), f[5], out=f)
  y = torch.zeros(3, 32, dtype=BF)
  with pytest.raises(ValueError, match="overlaps"):
    ops.mx_linear(ops.Microscaled(y.view(U8)[:, :32].contiguous().view(F8), torch.zeros(3, 1, dtype=U8)),
                  ops.Microscaled(y.view(U8).view(6, 32)[:, :16], torch.zeros(6, 1, dtype=U8)), out=y[:, :6])


def test_gradients_and_tangents_are_refused():
  q = torch.zeros(6, 4, 32, dtype=BF, requires_grad=True)
  with pytest.raises(ValueError, match="no backward pass"):
    ops.paged_attention(**attention_args(q=q))
  k = torch.zeros(6, 2, 32, dtype=BF, requires_grad=True)
  with pytest.raises(ValueError, match="no backward pass"):
    ops.paged_cache_write(**write_args(k=k))
  x = torch.zeros(2, 32, requires_grad=True)
  for call in (lambda: ops.add_rms_norm(x, None, None), lambda: ops.add_rms_norm(x.detach(), x, None), lambda: ops.mx_quantize(x),
               lambda: ops.add_rms_norm(x.detach(), None, torch.ones(32, requires_grad=True)),
               lambda: ops.mx_linear(mx(2, 32), mx(3, 32), torch.zeros(3, requires_grad=True))):
    with pytest.raises(ValueError, match="no backward pass"):
      call()
  codes = ops.Microscaled(torch.zeros(2, 32).to(F8).requires_grad_(), torch.zeros(2, 1, dtype=U8))
  for call in (lambda: ops.mx_dequantize(codes), lambda: ops.mx_linear(codes, mx(3, 32)), lambda: ops.mx_linear(mx(3, 32), codes)):
    with pytest.raises(ValueError, match="no backward pass"):
      call()
  with torch.no_grad(), pytest.raises(_Launched):
    ops.mx_quantize(x)
  import torch.autograd.forward_ad as fwd
  with fwd.dual_level():
    d = fwd.make_dual(torch.zeros(2, 32), torch.ones(2, 32))
    with pytest.raises(ValueError, match="forward-mode"):
      ops.mx_quantize(d)


# ---- microscaled numbers and the norm ------------------------------------------------------

def mx(R, K, eight=True):
  return ops.Microscaled(torch.zeros(R, K, dtype=U8).view(F8) if eight else torch.zeros(R, K // 2, dtype=U8), torch.zeros(R, K // 32, dtype=U8))


@pytest.mark.parametrize("x,format,match", [
    (torch.zeros(2, 33), "mxfp8", "multiple of 32"), (torch.zeros(2, 0), "mxfp8", "multiple of 32"), (torch.zeros(()), "mxfp8", "multiple of 32"),
    (torch.zeros(2, 32), "mxfp6", "format"), (torch.zeros(2, 32, dtype=torch.float64), "mxfp4", "bfloat16"), (torch.zeros(2, 32, dtype=I32), "mxfp4", "bfloat16"),
])
def test_quantize_refuses(x, format, match):
  with pytest.raises(ValueError, match=match):
    ops.mx_quantize(x, format)


@pytest.mark.parametrize("x,match", [
    (ops.Microscaled(torch.zeros(2, 32), torch.zeros(2, 1, dtype=U8)), "codes"),
    (ops.Microscaled(torch.zeros(2, 16, dtype=U8), torch.zeros(2, 1)), "scales"),
    (ops.Microscaled(torch.zeros(2, 16, dtype=U8), torch.zeros(2, 2, dtype=U8)), "block of 32"),
    (ops.Microscaled(torch.zeros(2, 15, dtype=U8), torch.zeros(2, 1, dtype=U8)), "block of 32"),
    (ops.Microscaled(torch.zeros(2, 16, dtype=U8), torch.zeros(3, 1, dtype=U8)), "block of 32"),
    (ops.Microscaled(torch.zeros(2, 0, dtype=U8), torch.zeros(2, 0, dtype=U8)), "block of 32"),
])
def test_codes_and_scales_are_checked(x, match):
  with pytest.raises(ValueError, match=match):
    ops.mx_dequantize(x)
  with pytest.raises(ValueError, match=match):
    ops.mx_linear(x, mx(3, 32))
  with pytest.raises(ValueError, match=match):
    ops.mx_linear(mx(3, 32), x)


@pytest.mark.parametrize("shape", [(), (16,)])
def test_scales_without_a_dim(shape):
  x = ops.Microscaled(torch.zeros(shape, dtype=U8), torch.zeros((), dtype=U8))
  for call in (lambda: ops.mx_dequantize(x), lambda: ops.mx_linear(x, mx(3, 32, False))):
    with pytest.raises(ValueError, match="block of 32"):
      call()


@pytest.mark.parametrize("x,w,kw,match", [
    (mx(2, 64), mx(3, 32), {}, "against"), (mx(2, 32, False), mx(3, 32), {}, "4-bit x"), (mx(2, 32), mx(3, 32), dict(dtype=torch.float32), "dtype"),
    (mx(2, 32), mx(3, 32), dict(bias=torch.zeros(4)), "bias"), (mx(2, 32), mx(0, 32), {}, "against"),
    (mx(2, 32), mx(3, 32), dict(out=torch.zeros(2, 4, dtype=BF)), "out must be"), (mx(2, 32), mx(3, 32), dict(out=torch.zeros(2, 3)), "out must be"),
    (mx(2, 32), mx(3, 32), dict(out=torch.zeros(3, 2, dtype=BF).t()), "out must be"),
    (mx(2, 32), mx(3, 32), dict(out=torch.zeros(1, 3, dtype=BF).expand(2, 3)), "once"),
    (mx(2, 32), ops.Microscaled(torch.zeros(1, 3, 32, dtype=U8).view(F8), torch.zeros(1, 3, 1, dtype=U8)), {}, "features"),
])
def test_linear_refuses(x, w, kw, match):
  with pytest.raises(ValueError, match=match):
    ops.mx_linear(x, w, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(residual=torch.zeros(2, 64)), "one type"), (dict(residual=torch.zeros(3, 64, dtype=BF)), "shape"), (dict(x=torch.zeros(2, 64, dtype=torch.float64)), "bfloat16"),
    (dict(x=torch.zeros(2, 0, dtype=BF), residual=None), "\\[\\.\\.\\., C\\]"), (dict(weight=torch.zeros(32)), "weight"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(eps=math.inf), "eps"), (dict(output="fp8"), "output"), (dict(output="mxfp8", x=torch.zeros(2, 40, dtype=BF), residual=None, weight=None), "multiple of 32"),
    (dict(output="mxfp8", out=torch.zeros(2, 64, dtype=BF)), "without output"), (dict(residual=None, out_sum=torch.zeros(2, 64, dtype=BF)), "with a residual"),
    (dict(out=torch.zeros(2, 64)), "out must be"), (dict(out_sum=torch.zeros(3, 64, dtype=BF)), "out_sum must be"), (dict(out=torch.zeros(64, 2, dtype=BF).t()), "unit last"),
    (dict(out=torch.zeros(1, 64, dtype=BF).expand(2, 64)), "once"), (dict(output="mxfp4", out_sum=torch.zeros(2, 68, dtype=BF)[:, :64]), "16-byte"),
])
def test_norm_refuses(kw, match):
  a = dict(x=torch.zeros(2, 64, dtype=BF), residual=torch.zeros(2, 64, dtype=BF), weight=torch.ones(64))
  a.update(kw)
  with pytest.raises(ValueError, match=match):
    ops.add_rms_norm(**a)


# ---- the C calls --------------------------------------------------------------------------

@pytest.fixture
def lib():
  return _lib.load()


def c_attention(**kw):
  a = _lib.PagedAttentionArgs(B=2, H=4, Hkv=2, D=64, Tq=6, pages=5, page_rows=16, table_cols=3, scale=0.125, causal=1, q=4096, k=4096, v=4096, out=4096, cu_q=4096,
                              len_k=4096, table=4096, table_s=3)
  a.q_s[:], a.o_s[:] = (256, 64), (256, 64)
  a.k_s[:], a.v_s[:] = (2048, 128, 64), (2048, 128, 64)
  for k, v in kw.items():
    if isinstance(v, tuple):
      getattr(a, k)[:] = v
    else:
      setattr(a, k, v)
  return a


@pytest.mark.parametrize("kw,match", [
    (dict(B=0), "sizes"), (dict(H=5), "evenly"), (dict(D=60), "head dim"), (dict(D=136), "head dim"), (dict(dtype=2), "type"), (dict(scale=math.nan), "scale"),
    (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"), (dict(page_rows=8), "pages"), (dict(page_rows=24), "pages"), (dict(table_cols=0), "pages"),
    (dict(table_cols=1 << 27), "2\\^30"), (dict(k=None), "non-null"), (dict(table=None), "non-null"), (dict(len_k=None), "non-null"), (dict(cu_q=None), "non-null"),
    (dict(k=4104), "aligned"), (dict(out=4104), "aligned"), (dict(k_s=(2048, 128, 60)), "multiples of 8"), (dict(k_s=(2048, 56, 64)), "strides"),
    (dict(v_s=(2048, 1 << 24, 64)), "strides"), (dict(v_s=(-8, 128, 64)), "strides"), (dict(q_s=(250, 64)), "multiples of 8"), (dict(Tq=1 << 30), "2\\^30"),
])
def test_c_attention_refuses(lib, kw, match):
  a = c_attention(**kw)
  assert lib.sf_hip_paged_attention_fwd(C.byref(a), None, 0, None) != 0
  assert __import__("re").search(match, _lib.last_error())
  assert lib.sf_hip_paged_attention_workspace_bytes(C.byref(a)) == 0


def test_c_attention_workspace(lib):
  assert lib.sf_hip_paged_attention_fwd(C.byref(c_attention(Tq=0)), None, 0, None) == 0
  a = c_attention(Tq=2, table_cols=4096)                       # long caches: slices are joined through a workspace
  need = lib.sf_hip_paged_attention_workspace_bytes(C.byref(a))
  assert need > 0
  assert lib.sf_hip_paged_attention_fwd(C.byref(a), None, 0, None) != 0 and "workspace" in _lib.last_error()
  assert lib.sf_hip_paged_attention_fwd(C.byref(a), 4096, need - 1, None) != 0 and "workspace" in _lib.last_error()
  for kw in (dict(Tq=600, table_cols=400), dict(B=200, Tq=200, table_cols=100), dict(B=1000, Tq=1000), dict(B=13, Tq=524, H=16, table_cols=188)):
    assert lib.sf_hip_paged_attention_workspace_bytes(C.byref(c_attention(**kw))) < 512 << 20


@pytest.mark.parametrize("kw,match", [
    (dict(B=0), "B=0"), (dict(D=60), "D=60"), (dict(T=-1), "T=-1"), (dict(T=(1 << 30) + 1), "T="), (dict(page_rows=8), "pages"), (dict(k=None), "non-null"), (dict(cu=None), "non-null"),
    (dict(k=4104), "aligned"), (dict(k_pages=4104), "aligned"), (dict(k_s=(60, 64)), "multiples of 8"), (dict(vp_s=(2048, 120, 60)), "strides"), (dict(len_k=None), "non-null"),
])
def test_c_write_refuses(lib, kw, match):
  a = _lib.PagedWriteArgs(B=2, Hkv=2, D=64, T=6, pages=5, page_rows=16, table_cols=3, k=4096, v=4096, k_pages=4096, v_pages=4096, cu=4096, len_k=4096, table=4096, table_s=3)
  a.k_s[:], a.v_s[:], a.kp_s[:], a.vp_s[:] = (128, 64), (128, 64), (2048, 128, 64), (2048, 128, 64)
  for k, v in kw.items():
    if isinstance(v, tuple):
      getattr(a, k)[:] = v
    else:
      setattr(a, k, v)
  assert lib.sf_hip_paged_write_fwd(C.byref(a), None) != 0
  assert match in _lib.last_error()


@pytest.mark.parametrize("kw,match", [
    (dict(K=33), "multiple of 32"), (dict(K=0), "multiple of 32"), (dict(R=-1), "multiple of 32"), (dict(format=2), "format"), (dict(dtype=3), "type"), (dict(x=None), "non-null"),
    (dict(codes=4104), "aligned"), (dict(x_rs=60), "aligned"), (dict(c_rs=40), "aligned"),
])
def test_c_convert_refuses(lib, kw, match):
  for fn in (lib.sf_hip_mx_encode_fwd, lib.sf_hip_mx_decode_fwd):
    a = _lib.MxConvertArgs(R=2, K=64, x=4096, x_rs=64, codes=4096, c_rs=64, scales=4096, s_rs=2)
    for k, v in kw.items():
      setattr(a, k, v)
    assert fn(C.byref(a), None) != 0 and match in _lib.last_error()


def c_norm(**kw):
  a = _lib.AddRmsNormArgs(R=2, C=64, eps=1e-6, x=4096, x_rs=64, y=4096, y_rs=64)
  for k, v in kw.items():
    setattr(a, k, v)
  return a


@pytest.mark.parametrize("kw,match", [
    (dict(C=0), "rows of 0"), (dict(R=-1), "rows"), (dict(dtype=3), "type"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(x=None), "non-null"), (dict(y=None), "non-null"),
    (dict(codes=4096, scales=4096), "either"), (dict(y=None, codes=4096), "non-null"), (dict(y=None, codes=4096, scales=4096, c_rs=64, format=2), "format"),
    (dict(y=None, codes=4096, scales=4096, c_rs=40), "multiple of 32"), (dict(y=None, codes=4096, scales=4096, c_rs=64, C=40), "multiple of 32"),
    (dict(y=None, codes=4096, scales=4096, c_rs=64, x=4100), "aligned"),
])
def test_c_norm_refuses(lib, kw, match):
  assert lib.sf_hip_add_rms_norm_fwd(C.byref(c_norm(**kw)), None) != 0
  assert match in _lib.last_error()


def c_linear(**kw):
  a = _lib.MxLinearArgs(M=200, N=300, K=256, x=4096, x_rs=256, x_scales=4096, xs_rs=8, w=4096, w_rs=256, w_scales=4096, ws_rs=8, y=4096, y_rs=300)
  for k, v in kw.items():
    setattr(a, k, v)
  return a


@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), "M=-1"), (dict(N=0), "N=0"), (dict(K=48), "K=48"), (dict(K=1 << 23), "K="), (dict(x_format=1), "formats"), (dict(w_format=2), "formats"), (dict(dtype=2), "type"),
    (dict(x=None), "non-null"), (dict(y=None), "non-null"), (dict(w=4104), "aligned"), (dict(x_rs=240), "row strides"), (dict(x_rs=1 << 23), "row strides"), (dict(ws_rs=7), "row strides"),
    (dict(y_rs=299), "row strides"),
])
def test_c_linear_refuses(lib, kw, match):
  a = c_linear(**kw)
  assert lib.sf_hip_mx_linear_fwd(C.byref(a), None, 0, None) != 0
  assert match in _lib.last_error()
  assert lib.sf_hip_mx_linear_workspace_bytes(C.byref(a)) == 0


def test_c_linear_workspace(lib):
  assert lib.sf_hip_mx_linear_workspace_bytes(C.byref(c_linear(M=8))) == 0
  a = c_linear(M=100, N=1024, K=8192, x_rs=8192, w_rs=8192, xs_rs=256, ws_rs=256, y_rs=1024)       # few tiles, long rows: k in parts
  need = lib.sf_hip_mx_linear_workspace_bytes(C.byref(a))
  assert need > 0 and need % (100 * 1024 * 4) == 0
  assert lib.sf_hip_mx_linear_fwd(C.byref(a), None, 0, None) != 0 and "workspace" in _lib.last_error()
  assert lib.sf_hip_mx_linear_fwd(C.byref(a), 4096, need - 16, None) != 0 and "workspace" in _lib.last_error()
  assert lib.sf_hip_mx_linear_fwd(C.byref(c_linear(M=0)), None, 0, None) == 0


@pytest.mark.parametrize("name", ["sf_paged_attention_args", "sf_paged_write_args", "sf_mx_convert_args", "sf_add_rms_norm_args", "sf_mx_linear_args"])
def test_filled_structs(name):
  """The packed form of a struct's fields is the struct."""
  S = _lib.STRUCTS[name]
  flat, n = [], 1
  for _, t in S._fields_:
    for _ in range(t._length_ if issubclass(t, C.Array) else 1):
      flat.append(n)
      n += 1
  a, i = _lib.filler(S)(*flat), 0
  for f, t in S._fields_:
    v = getattr(a, f)
    for x in (list(v) if issubclass(t, C.Array) else [v]):
      i += 1
      assert x == i, f


# ---- index arithmetic that the kernels restate ---------------------------------------------------------

@pytest.mark.parametrize("per", [1, 2, 3, 4, 5, 7, 8, 12, 63, 64, 65, 100, 1000, 4095, 1 << 20, (1 << 26) - 1, 1 << 26])
def test_page_of_a_unit(per):
  """page_div and page_of (csrc/packed.h): units of 16 rows below 2^27 over the units of a page, exactly; the multiplier fits 32 bits."""
  up = 0
  while (1 << up) < per:
    up += 1
  m, s = (1 << (31 + up)) // per + 1, 31 + up
  assert 0 < m < 1 << 32
  edge = [k * per + d for k in (0, 1, 2, 3, 17, (1 << 27) // per - 1, (1 << 27) // per) for d in (-1, 0, 1)]
  g = torch.Generator().manual_seed(per)
  for i in edge + [int(x) for x in torch.randint(0, 1 << 27, (2000,), generator=g)]:
    if 0 <= i < 1 << 27:
      assert (i * m) >> s == i // per


@pytest.mark.parametrize("KT,NT", [(64, 256), (64, 512), (64, 64), (32, 64)])
@pytest.mark.parametrize("DP", [32, 64, 96, 128])
def test_units_of_a_staged_tile(KT, NT, DP):
  """Stage of a paged cache (csrc/packed.h): every 16-byte piece of a tile is stored once, by a wave whose load of it lies in one page of a
  multiple of 16 rows, whatever tile and page."""
  if KT == 32 and DP <= 64:
    pytest.skip("tiles of 32 keys are for head dims above 64")
  pieces, waves = DP // 8, NT // 64
  RU = KT // waves if waves > KT // 16 else 16
  UN = KT // RU // waves
  LU = -(-RU * pieces // 64)
  stored = set()
  for wave in range(waves):
    for x in range(UN):
      first = wave * UN * RU + x * RU
      for rows in (16, 48, 64):
        for j0 in range(0, 10 * KT, KT):
          assert (j0 + first) // rows == (j0 + first + RU - 1) // rows
          unit = (j0 + first) >> 4
          page = unit // (rows // 16)
          assert page == (j0 + first) // rows and ((unit - page * (rows // 16)) << 4) + (first & 15) == (j0 + first) % rows
      for u in range(LU):
        for lane in range(64):
          idx = 64 * u + lane
          if idx < RU * pieces:
            at = (first + idx // pieces, idx % pieces)
            assert at not in stored
            stored.add(at)
  assert stored == {(k, p) for k in range(KT) for p in range(pieces)}


@pytest.mark.parametrize("K8", [(k, f) for k in range(512, 5000, 128) for f in (2, 4)])
def test_groups_of_scales_stay_in_their_rows(K8):
  """mx_linear_pp_kernel: 16 scales a copy, the last group ending with the row; a step's scales lie in its group's, at a whole word but for
  half a word of 64-k steps; a group's buffer is not written before its last step is read."""
  K, SB = K8
  blocks, n, GS = K // 32, K // (32 * SB), 16 // SB
  groups = -(-n // GS)
  at = lambda g: min(16 * g, blocks - 16)
  for t in range(n):
    g = t // GS
    first = SB * t - at(g)
    assert at(g) >= 0 and at(g) % 4 == 0 and at(g) + 16 <= blocks
    assert 0 <= first and first + SB <= 16 and (first % 4 == 0 or SB == 2)
  # steps in a row over tiles: group buffers in turn, copies three steps ahead
  first_of, last_of, total = {}, {}, 0
  for tile in range(3):
    for t in range(n):
      g = tile * groups + t // GS
      first_of.setdefault(g, total)
      last_of[g] = total
      total += 1
  for g in first_of:
    if g + 4 in first_of:
      assert first_of[g + 4] - 3 > last_of[g]


@pytest.mark.parametrize("pieces", [8, 4])
def test_lds_slots_are_a_permutation(pieces):
  """16 rows read together (one piece each) fall on 16 different 16-byte slots of 256 bytes, and a row's pieces on all of its slots."""
  slot = (lambda r, p: p ^ ((r >> 1) & 7)) if pieces == 8 else (lambda r, p: p ^ ((r >> 2) & 3))
  for r in range(128):
    assert {slot(r, p) for p in range(pieces)} == set(range(pieces))
  for r0 in range(0, 128, 16):
    for p in range(pieces):
      assert len({(r * pieces * 16 + slot(r, p) * 16) % 256 for r in range(r0, r0 + 16)}) == 16
  half = lambda r, p: (r >> 1) * 64 + (((2 * (r & 1) + p) ^ ((r >> 3) & 1)) << 4)       # rows of 32 bytes, two a line
  for r0 in range(0, 256, 16):
    for p in range(2):
      assert len({half(r, p) % 256 for r in range(r0, r0 + 16)}) == 16
  assert len({half(r, p) for r in range(256) for p in range(2)}) == 512


def test_host_module_does_nothing_of_other_forms(lib):
  """The host module answers None to host tensors, other objects and other numbers of arguments."""
  front = _lib.front(lib, ops.Microscaled)
  assert front is not None and front.abi_version == _lib.ABI_VERSION
  x = torch.zeros(2, 64, dtype=BF)
  pages = torch.zeros(5, 16, 2, 32, dtype=BF)
  for name, args in (("add_rms_norm", (x, x, None, 1e-6, None)), ("mx_quantize", (x, "mxfp8")), ("mx_linear", (*mx(2, 64), *mx(3, 64), None, BF)), ("mx_dequantize", (*mx(2, 64), BF)),
                     ("paged_cache_write", (torch.zeros(6, 2, 32, dtype=BF),) * 2 + (pages, pages.clone(), torch.zeros(2, 3, dtype=I32), ints(0, 2, 6), ints(20, 40), None)),
                     ("paged_attention", (torch.zeros(6, 4, 32, dtype=BF), pages, pages, torch.zeros(2, 3, dtype=I32), ints(0, 2, 6), ints(20, 40), None, True, None, None))):
    call = getattr(front, name)
    assert call(*args) is None and call(*args[:-1]) is None and call(*args, None) is None and call() is None
    for i in range(len(args)):
      for other in (None, 3, "x", x, object()):
        assert call(*args[:i], other, *args[i + 1:]) is None
  for args in ((), (1,) * 9, (0,) * 9 + (object,), ("a",) * 9 + (object,)):
    with pytest.raises((TypeError, ValueError)):
      front.bind(*args)


def test_without_the_host_module(monkeypatch, lib):
  monkeypatch.setattr(_lib, "front_path", lambda: _lib.LIB_PATH.with_name("absent.so"))
  assert _lib.front(lib, ops.Microscaled) is None


@pytest.mark.parametrize("gx,gy", [(1, 1025), (1030, 1), (9, 131), (40, 32), (63, 64), (129, 8), (33, 33), (7, 300)])
def test_bands_reach_every_tile_once(gx, gy):
  """mx_tile_kernel's order of tiles beyond 1024 of them."""
  total, band_rows, seen = gx * gy, 8, set()
  for i in range(total):
    t = (i & 7) * (total >> 3) + min(i & 7, total & 7) + (i >> 3)
    band = t // (band_rows * gy)
    q, bh = t - band * band_rows * gy, min(band_rows, gx - band * band_rows)
    by = q // bh
    bx = band * band_rows + q - by * bh
    assert 0 <= bx < gx and 0 <= by < gy
    seen.add((bx, by))
  assert len(seen) == total
