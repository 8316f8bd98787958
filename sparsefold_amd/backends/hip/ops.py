"""Tensor-level wrappers over the C ABI (include/sparsefold_hip.h).

Each wrapper checks devices, shapes and dtypes in Python (ValueError, as the reference's
native wrappers do, ``backends/vecops/kernels/registry.py:2910-2929``), allocates outputs and
workspaces with torch on the input's device, and launches on torch's current HIP stream.
Nothing here computes on the host: every numeric result comes from libsparsefold_hip.
"""
from __future__ import annotations

import ctypes as C
import itertools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from sparsefold_amd import _lib

BF16 = torch.bfloat16


# The small calls are bound by this file: a call of 20 residues spends longer here than its kernels
# run.  Pointers and streams are passed as plain ints (every struct field and argument that takes one
# is declared c_void_p), the device check reads ints, and messages are formatted only when raised.
def _vp(t: torch.Tensor | None):
  return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t: torch.Tensor):
  """torch's current stream on t's device (the raw handle; the public accessor builds a Stream
  object per call, which costs more than some of the kernels it launches)."""
  if _raw_stream is not None:
    return _raw_stream(t.get_device())
  return torch.cuda.current_stream(t.device).cuda_stream


def _require_cuda(*ts: torch.Tensor | None) -> torch.device:
  first, index = None, -1
  for t in ts:
    if t is None:
      continue
    i = t.get_device()                                         # (-1 on the host)
    if i != index or i < 0:
      if not t.is_cuda:
        raise ValueError(f"HIP kernels need device tensors, got a tensor on {t.device}")
      if first is not None:
        raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
      first, index = t, i
  if first is None:
    raise ValueError("no device tensor given")
  return first.device


def _require(cond: bool, msg: str) -> None:
  if not cond:
    raise ValueError(msg)


def _bf16(t: torch.Tensor) -> torch.Tensor:
  return t if t.dtype == BF16 else t.to(BF16)


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
  return None if t is None else t.to(torch.float32).contiguous()


def _u8(t: torch.Tensor) -> torch.Tensor:
  """Byte mask: a bool tensor is reinterpreted in place (torch stores bool as 0/1 bytes)."""
  if t.dtype == torch.uint8:
    return t
  if t.dtype == torch.bool:
    return t.view(torch.uint8)
  return (t != 0).view(torch.uint8)


def _rows(t: torch.Tensor, last: int) -> torch.Tensor:
  """2-D row view ``[M, last]`` with unit last stride and 16-byte aligned rows."""
  t2 = t.reshape(-1, last)
  if t2.stride(-1) != 1 or t2.stride(0) % 8 != 0 or t2.data_ptr() % 16 != 0:
    t2 = t2.contiguous()
  return t2


# ---------------------------------------------------------------------------------------
# attention core
# ---------------------------------------------------------------------------------------

def attention(q, k, v, *, scale: float, bias=None, mask_q=None, mask_k=None, gate=None, out=None,
              schedule: int = 0):
  """Core launch on 2-level batched views.

  q ``[B0,B1,Q,H,D]``, k ``[B0,B1,K,H,D]``, v ``[B0,B1,K,H,Dv]``, gate like the output
  ``[B0,B1,Q,H,Dv]``; bias ``[B0,B1,H,Q,K]`` (zero strides allowed), masks ``[B0,B1,Q]`` /
  ``[B0,B1,K]`` uint8.  All bf16 with unit last stride.  ``schedule``: 0 chooses the work
  decomposition from the sizes, 1 / 2 force shared-tile / per-wave tasks, 3 the shared-bias
  kernel (5 samples, head dim 48, one bias for all samples; refused otherwise).  Returns ``out``.
  """
  dev = _require_cuda(q, k, v, bias, mask_q, mask_k, gate, out)
  _require(q.ndim == 5 and k.ndim == 5 and v.ndim == 5, "attention: q/k/v must be [B0,B1,L,H,D]")
  B0, B1, Q, H, D = q.shape
  K, Dv = k.shape[2], v.shape[-1]
  _require(tuple(k.shape) == (B0, B1, K, H, D), f"attention: k shape {tuple(k.shape)} vs q {tuple(q.shape)}")
  _require(tuple(v.shape[:4]) == (B0, B1, K, H), f"attention: v shape {tuple(v.shape)}")
  for name, t in (("q", q), ("k", k), ("v", v), ("gate", gate), ("bias", bias)):
    if t is not None:
      _require(t.dtype == BF16, f"attention: {name} must be bfloat16, got {t.dtype}")
      _require(t.stride(-1) == 1, f"attention: {name} needs a unit last stride")
  if out is None:
    out = torch.empty((B0, B1, Q, H, Dv), dtype=BF16, device=dev)
  _require(tuple(out.shape) == (B0, B1, Q, H, Dv) and out.stride(-1) == 1, "attention: bad out")
  a = _lib.AttentionArgs()
  a.B0, a.B1, a.Q, a.K, a.H, a.D, a.Dv = B0, B1, Q, K, H, D, Dv
  a.scale = float(scale)
  a.q, a.q_s = _vp(q), (C.c_int64 * 4)(*q.stride()[:4])
  a.k, a.k_s = _vp(k), (C.c_int64 * 4)(*k.stride()[:4])
  a.v, a.v_s = _vp(v), (C.c_int64 * 4)(*v.stride()[:4])
  if bias is not None:
    _require(tuple(bias.shape) == (B0, B1, H, Q, K), f"attention: bias shape {tuple(bias.shape)}")
    a.bias, a.bias_s = _vp(bias), (C.c_int64 * 4)(*bias.stride()[:4])
  if mask_q is not None:
    _require(tuple(mask_q.shape) == (B0, B1, Q) and mask_q.dtype == torch.uint8, "attention: bad mask_q")
    a.mask_q, a.mq_s = _vp(mask_q), (C.c_int64 * 3)(*mask_q.stride())
  if mask_k is not None:
    _require(tuple(mask_k.shape) == (B0, B1, K) and mask_k.dtype == torch.uint8, "attention: bad mask_k")
    a.mask_k, a.mk_s = _vp(mask_k), (C.c_int64 * 3)(*mask_k.stride())
  if gate is not None:
    _require(tuple(gate.shape) == (B0, B1, Q, H, Dv), f"attention: gate shape {tuple(gate.shape)}")
    a.gate, a.g_s = _vp(gate), (C.c_int64 * 4)(*gate.stride()[:4])
  a.out, a.o_s = _vp(out), (C.c_int64 * 4)(*out.stride()[:4])
  _require(schedule in (0, 1, 2, 3), f"attention: schedule {schedule} is not 0, 1, 2 or 3")
  a.schedule = schedule
  lib = _lib.load()
  _lib.check(lib.sf_hip_attention_fwd(C.byref(a), _stream(q)), "sf_hip_attention_fwd")
  return out


# ---------------------------------------------------------------------------------------
# row kernels
# ---------------------------------------------------------------------------------------

def layer_norm(x: torch.Tensor, gamma=None, beta=None, *, eps: float = 1e-5, scale=None, shift=None):
  """LN over the last dim (bf16 in / out).  With ``scale``/``shift`` ([R, C] bf16) this is
  the AdaLN modulation, row m using condition row ``m % R``."""
  _require_cuda(x, gamma, beta, scale, shift)
  Cn = x.shape[-1]
  x2 = _rows(_bf16(x), Cn)
  y = torch.empty(x2.shape, dtype=BF16, device=x.device)
  a = _lib.LayerNormArgs()
  a.M, a.C, a.eps = x2.shape[0], Cn, float(eps)
  a.x, a.x_rs = _vp(x2), x2.stride(0)
  g, b = _f32(gamma), _f32(beta)
  a.gamma, a.beta = _vp(g), _vp(b)
  if scale is not None:
    s2, h2 = _rows(_bf16(scale), Cn), _rows(_bf16(shift), Cn)
    _require(s2.shape == h2.shape, "layer_norm: scale/shift shapes differ")
    a.scale, a.shift, a.cond_rows, a.cond_rs = _vp(s2), _vp(h2), s2.shape[0], s2.stride(0)
  a.y, a.y_rs = _vp(y), y.stride(0)
  _lib.check(_lib.load().sf_hip_layer_norm_fwd(C.byref(a), _stream(x)), "sf_hip_layer_norm_fwd")
  return y.view(*x.shape[:-1], Cn)


def linear(x: torch.Tensor, wt: torch.Tensor, bias=None, *, residual=None, mul=None,
           post_sigmoid: bool = False, ycols: int | None = None, yt=None, tcol0: int = 0,
           want_y: bool = True):
  """``post(x @ wt.T + bias) * mul + residual`` with ``wt`` ``[N, K]`` bf16 (K contiguous).

  ``mul`` ``[R, N]`` multiplies row m by ``mul[m % R]``.  ``yt`` (``[T, M]`` bf16) receives
  columns ``[tcol0, tcol0+T)`` transposed.  Returns ``y`` ``[..., ycols or N]`` or None."""
  _require_cuda(x, wt, bias, residual, mul, yt)
  N, K = wt.shape
  _require(x.shape[-1] == K, f"linear: x last dim {x.shape[-1]} != weight K {K}")
  _require(K % 8 == 0, "linear: K must be a multiple of 8")
  _require(wt.dtype == BF16 and wt.is_contiguous(), "linear: wt must be contiguous bf16 [N, K]")
  x2 = _rows(_bf16(x), K)
  M = x2.shape[0]
  a = _lib.LinearArgs()
  a.M, a.N, a.K = M, N, K
  a.x, a.x_rs, a.wt = _vp(x2), x2.stride(0), _vp(wt)
  bias_f = _f32(bias)
  a.bias = _vp(bias_f)
  ycols = N if ycols is None else ycols
  y = None
  if want_y:
    y = torch.empty((M, ycols), dtype=BF16, device=x.device)
    a.y, a.y_rs, a.ycols = _vp(y), y.stride(0), ycols
  if residual is not None:
    r2 = _bf16(residual).reshape(M, -1)
    _require(r2.shape[1] == ycols and r2.stride(-1) == 1, "linear: residual shape")
    a.residual, a.r_rs = _vp(r2), r2.stride(0)
  if mul is not None:
    m2 = _bf16(mul).reshape(-1, N)
    _require(m2.stride(-1) == 1, "linear: mul needs a unit last stride")
    a.mul, a.mul_rows, a.mul_rs = _vp(m2), m2.shape[0], m2.stride(0)
  else:
    a.mul_rows = 1
  a.post_sigmoid = int(bool(post_sigmoid))
  if yt is not None:
    _require(yt.dtype == BF16 and yt.shape[-1] == M and yt.stride(-1) == 1, "linear: yt shape")
    a.tcol0, a.tcols, a.yt, a.yt_rs = tcol0, yt.shape[0], _vp(yt), yt.stride(0)
  _lib.check(_lib.load().sf_hip_linear_fwd(C.byref(a), _stream(x)), "sf_hip_linear_fwd")
  return None if y is None else y.view(*x.shape[:-1], ycols)


def pair_logits(z: torch.Tensor, ln_w, ln_b, w_t: torch.Tensor, *, seg: int = 0, group: int = 0) -> torch.Tensor:
  """``[..., C]`` pair activations -> LN + projection logits planes.

  ``seg == 0``: ``[H, P]``.  ``seg > 0``: ``[H // group, P // seg, group, seg]`` (plane
  ``blk * group + h``, position ``u * seg + r``), the CrossAttTransformer pack layout."""
  _require_cuda(z, ln_w, ln_b, w_t)
  H, Cn = w_t.shape
  z2 = _rows(_bf16(z), Cn)
  P = z2.shape[0]
  _require(z2.stride(0) == Cn, "pair_logits: z rows must be contiguous")
  if seg:
    _require(P % seg == 0 and group > 0 and H % group == 0, "pair_logits: P % seg and H % group must be 0")
    out = torch.empty((H // group, P // seg, group, seg), dtype=BF16, device=z.device)
  else:
    out = torch.empty((H, P), dtype=BF16, device=z.device)
  lw, lb = _f32(ln_w), _f32(ln_b)
  wt = _bf16(w_t).contiguous()
  a = _lib.PairLogitsArgs()
  a.P, a.C, a.H = P, Cn, H
  a.z, a.ln_w, a.ln_b, a.w_t, a.out = _vp(z2), _vp(lw), _vp(lb), _vp(wt), _vp(out)
  a.seg, a.group = int(seg), int(group) if seg else 0
  _lib.check(_lib.load().sf_hip_pair_logits_fwd(C.byref(a), _stream(z)), "sf_hip_pair_logits_fwd")
  return out


def window_gather(src: torch.Tensor, idx: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
  """``src [S, rows, C]`` -> ``[S, UK, C]`` by flat index ``idx [UK]`` (masked -> 0)."""
  _require_cuda(src, idx, mask)
  S, rows, Cn = src.shape
  src = _bf16(src).contiguous()
  idx32 = idx.reshape(-1).to(torch.int32).contiguous()
  m8 = _u8(mask.reshape(-1)).contiguous()
  _require(idx32.numel() == m8.numel(), "window_gather: idx / mask sizes differ")
  UK = idx32.numel()
  keys = torch.empty((S, UK, Cn), dtype=BF16, device=src.device)
  a = _lib.WindowGatherArgs()
  a.S, a.rows, a.C, a.UK = S, rows, Cn, UK
  a.src, a.idx, a.mask, a.keys = _vp(src), _vp(idx32), _vp(m8), _vp(keys)
  _lib.check(_lib.load().sf_hip_window_gather_fwd(C.byref(a), _stream(src)), "sf_hip_window_gather_fwd")
  return keys


# ---------------------------------------------------------------------------------------
# triangle attention module
# ---------------------------------------------------------------------------------------

def triangle_workspace_bytes(N: int, C_: int, H: int, D: int) -> int:
  return int(_lib.load().sf_hip_triangle_workspace_bytes(N, C_, H, D))


def triangle_attention(z: torch.Tensor, seq_mask: torch.Tensor, ln_w, ln_b, w_qkvgb: torch.Tensor,
                       w_o: torch.Tensor, *, num_head: int, transpose: bool, add_residual: bool = True,
                       workspace: torch.Tensor | None = None, stages: int = _lib.TRI_STAGE_ALL,
                       out: torch.Tensor | None = None, fixup_sum_limit: float = 0.0) -> torch.Tensor:
  """GridSelfAttention on ``z [N, N, C]`` (bf16).  Weights packed as the C ABI documents.
  ``stages`` selects a subset of the pipeline (projection / attention / output projection)
  against a caller-held ``workspace``.  ``fixup_sum_limit`` > 0 lowers the weight-sum limit
  above which a (row, head) is recomputed by the exact two-pass softmax (0 = the default 2^100)."""
  _require_cuda(z, seq_mask, ln_w, ln_b, w_qkvgb, w_o, workspace)
  if not (z.ndim == 3 and z.shape[0] == z.shape[1]):
    raise ValueError(f"triangle: z must be [N, N, C], got {tuple(z.shape)}")
  N, _, Cn = z.shape
  HD = w_o.shape[1]
  _require(HD % num_head == 0, "triangle: output projection width not divisible by heads")
  D = HD // num_head
  if w_qkvgb.shape != (4 * HD + num_head, Cn):
    raise ValueError(f"triangle: w_qkvgb shape {tuple(w_qkvgb.shape)}")
  if w_o.shape != (Cn, HD):
    raise ValueError(f"triangle: w_o shape {tuple(w_o.shape)}")
  _require(seq_mask.shape == (N,), "triangle: seq_mask must be [N]")
  zc = _bf16(z).contiguous()
  m8 = _u8(seq_mask).contiguous()
  lw, lb = _f32(ln_w), _f32(ln_b)
  need = triangle_workspace_bytes(N, Cn, num_head, D)
  if workspace is None or workspace.numel() < need:
    workspace = torch.empty(need, dtype=torch.uint8, device=z.device)
  if out is None:
    out = torch.empty_like(zc)
  a = _lib.TriangleArgs()
  a.N, a.C, a.H, a.D = N, Cn, num_head, D
  a.transpose, a.add_residual = int(bool(transpose)), int(bool(add_residual))
  a.z, a.seq_mask, a.ln_w, a.ln_b = _vp(zc), _vp(m8), _vp(lw), _vp(lb)
  a.w_qkvgb, a.w_o, a.out = _vp(w_qkvgb), _vp(w_o), _vp(out)
  _require(fixup_sum_limit >= 0.0, "triangle: fixup_sum_limit must be >= 0")
  a.fixup_sum_limit = float(fixup_sum_limit)
  if stages == _lib.TRI_STAGE_ALL:
    rc = _lib.load().sf_hip_triangle_attn_fwd(C.byref(a), _vp(workspace), workspace.numel(), _stream(z))
  else:
    rc = _lib.load().sf_hip_triangle_stage_fwd(C.byref(a), stages, _vp(workspace), workspace.numel(), _stream(z))
  _lib.check(rc, "sf_hip_triangle_attn_fwd")
  return out


# per-call seeds of the block sampler when the caller gives none (the reference draws them from a
# process-wide counter, backends/vecops/kernels/registry.py:3033)
_ibs_seed_counter = itertools.count()


def triangle_ibs_workspace_bytes(N: int, C_: int, H: int, D: int) -> int:
  return int(_lib.load().sf_hip_triangle_ibs_workspace_bytes(N, C_, H, D))


def triangle_attention_ibs(z: torch.Tensor, seq_mask: torch.Tensor, ln_w, ln_b, w_qkvgb: torch.Tensor,
                           w_o: torch.Tensor, *, num_head: int, transpose: bool, num_samples: int,
                           num_rand_blocks: int, t_prob: float, tr_prob: float, u_prob: float,
                           index_map: torch.Tensor | None = None, weight_map: torch.Tensor | None = None,
                           seed: int | None = None, add_residual: bool = True,
                           workspace: torch.Tensor | None = None, out: torch.Tensor | None = None,
                           fixup_sum_limit: float = 0.0):
  """GridSelfAttention on ``z [N, N, C]`` with block-sparse (IBS) attention rows; returns
  ``(out, index_map, weight_map)``, maps int32 / float32 ``[N, H, ceil(N/32), num_samples]``.
  Given maps (both or neither, as backends/vecops/kernels/registry.py:2985-3002 requires) are
  reused; otherwise they are sampled with ``seed`` (default: the next value of a process-wide
  counter).  ``fixup_sum_limit`` > 0 lowers the weight-sum limit above which a (row, head) is
  recomputed by the exact block-sparse kernel (0 = the default 2^100)."""
  _require_cuda(z, seq_mask, ln_w, ln_b, w_qkvgb, w_o, workspace, index_map, weight_map)
  _require(fixup_sum_limit >= 0.0, "triangle_ibs: fixup_sum_limit must be >= 0")
  _require(z.ndim == 3 and z.shape[0] == z.shape[1], f"triangle_ibs: z must be [N, N, C], got {tuple(z.shape)}")
  _require((index_map is None) == (weight_map is None), "index_map and weight_map must be both present or both omitted")
  N, _, Cn = z.shape
  HD = w_o.shape[1]
  _require(HD % num_head == 0, "triangle_ibs: output projection width not divisible by heads")
  D = HD // num_head
  _require(tuple(w_qkvgb.shape) == (4 * HD + num_head, Cn), f"triangle_ibs: w_qkvgb shape {tuple(w_qkvgb.shape)}")
  _require(tuple(w_o.shape) == (Cn, HD), f"triangle_ibs: w_o shape {tuple(w_o.shape)}")
  _require(seq_mask.shape == (N,), "triangle_ibs: seq_mask must be [N]")
  need = triangle_ibs_workspace_bytes(N, Cn, num_head, D)
  _require(need > 0, f"triangle_ibs: unsupported sizes N={N} C={Cn} H={num_head} D={D} "
           "(block-sparse rows need C = 128, H = 4, D = 32, N <= 8192)")
  T = (N + 31) // 32
  shape = (N, num_head, T, int(num_samples))
  generate = index_map is None
  if generate:
    index_map = torch.empty(shape, dtype=torch.int32, device=z.device)
    weight_map = torch.empty(shape, dtype=torch.float32, device=z.device)
  else:
    _require(tuple(index_map.shape) == shape and tuple(weight_map.shape) == shape,
             f"triangle_ibs: maps must be {shape}, got {tuple(index_map.shape)} / {tuple(weight_map.shape)}")
    _require(index_map.dtype == torch.int32 and weight_map.dtype == torch.float32,
             "triangle_ibs: index_map int32 and weight_map float32")
    index_map, weight_map = index_map.contiguous(), weight_map.contiguous()
  zc = _bf16(z).contiguous()
  m8 = _u8(seq_mask).contiguous()
  lw, lb = _f32(ln_w), _f32(ln_b)
  if workspace is None or workspace.numel() < need:
    workspace = torch.empty(need, dtype=torch.uint8, device=z.device)
  if out is None:
    out = torch.empty_like(zc)
  a = _lib.TriangleArgs()
  a.N, a.C, a.H, a.D = N, Cn, num_head, D
  a.transpose, a.add_residual = int(bool(transpose)), int(bool(add_residual))
  a.z, a.seq_mask, a.ln_w, a.ln_b = _vp(zc), _vp(m8), _vp(lw), _vp(lb)
  a.w_qkvgb, a.w_o, a.out = _vp(w_qkvgb), _vp(w_o), _vp(out)
  a.fixup_sum_limit = float(fixup_sum_limit)
  p = _lib.IbsArgs()
  p.num_samples, p.num_rand_blocks = int(num_samples), int(num_rand_blocks)
  p.t_prob, p.tr_prob, p.u_prob = float(t_prob), float(tr_prob), float(u_prob)
  p.generate_maps = int(generate)
  p.seed = (next(_ibs_seed_counter) if seed is None else int(seed)) & ((1 << 64) - 1)
  p.index_map, p.weight_map = _vp(index_map), _vp(weight_map)
  rc = _lib.load().sf_hip_triangle_attn_ibs_fwd(C.byref(a), C.byref(p), _vp(workspace), workspace.numel(), _stream(z))
  _lib.check(rc, "sf_hip_triangle_attn_ibs_fwd")
  return out, index_map, weight_map


def default_scale(d: int) -> float:
  return 1.0 / math.sqrt(d)


# ---------------------------------------------------------------------------------------
# whole attention modules (one C call each; see sf_hip_self_attention_fwd /
# sf_hip_cross_attention_fwd)
# ---------------------------------------------------------------------------------------

def _u8_or_none(t):
  return None if t is None else _u8(t).contiguous()


def self_attention_module(x: torch.Tensor, mask, bias, cond, w: dict, *, num_head: int, head_dim: int,
                          add_residual: bool = True, pre=None, noalloc: bool = False) -> torch.Tensor:
  """SelfAttention.forward as one call.  ``x`` ``[..., N, C]`` (leading dims = samples),
  ``mask`` ``[N]`` or None, ``bias`` ``[H, N, N]`` (shared) or ``[S, H, N, N]`` or None,
  ``cond`` ``[N, Cs]`` or None; ``w`` holds the packed weights (keys as in the C struct).
  ``pre`` = (scale, shift, zgate) ``[N, C]`` views with one row stride (one layer of
  ``diffusion_conditioning``) replaces the AdaLN computation from ``cond``.  ``noalloc`` runs
  the allocation-free entry point (the library's fixed per-GPU scratch; no workspace)."""
  _require_cuda(x, mask, bias, cond, *(pre or ()))
  N, Cn = x.shape[-2], x.shape[-1]
  S = x.numel() // max(N * Cn, 1)
  H, D = num_head, head_dim
  x3 = _bf16(x).reshape(S, N, Cn).contiguous()
  out = torch.empty_like(x3)
  a = _lib.SelfAttentionArgs()
  a.S, a.N, a.C, a.H, a.D = S, N, Cn, H, D
  a.scale, a.add_residual = 0.0, int(bool(add_residual))
  a.x, a.out = _vp(x3), _vp(out)
  m8 = _u8_or_none(mask)
  a.mask = _vp(m8)
  if bias is not None:
    b = _bf16(bias)
    _require(b.stride(-1) == 1, "self_attention: bias keys must be contiguous")
    if b.dim() == 3:
      a.bias_s[0], a.bias_s[1], a.bias_s[2] = 0, b.stride(0), b.stride(1)
    else:
      a.bias_s[0], a.bias_s[1], a.bias_s[2] = b.stride(0), b.stride(1), b.stride(2)
    a.bias = _vp(b)
  c2 = None
  if cond is not None:
    c2 = _bf16(cond).contiguous()
    a.cond, a.Cs = _vp(c2), c2.shape[-1]
  for key in ("ln_w", "ln_b", "lnc_w", "lnc_b", "w_scale", "b_scale", "w_shift", "w_qkvg", "b_qkvg",
              "w_t2", "w_zc", "b_zc"):
    setattr(a, key, _vp(w.get(key)))
  if pre is not None:
    ps, pb, pz = pre
    rs = ps.stride(0)
    for t in pre:
      _require(t.dtype == torch.bfloat16 and tuple(t.shape) == (N, Cn) and t.stride() == (rs, 1),
               "self_attention: precomputed conditioning must be bf16 [N, C] views with one row stride")
    a.pre_scale, a.pre_shift, a.pre_zgate, a.pre_rs = _vp(ps), _vp(pb), _vp(pz), rs
  lib = _lib.load()
  if noalloc:      # the library's fixed per-GPU scratch instead of a workspace
    _lib.check(lib.sf_hip_self_attention_fwd_noalloc(C.byref(a), _stream(x)), "sf_hip_self_attention_fwd_noalloc")
    return out.view(x.shape)
  ws = torch.empty(int(lib.sf_hip_self_attention_workspace_bytes(C.byref(a))), dtype=torch.uint8, device=x.device)
  _lib.check(lib.sf_hip_self_attention_fwd(C.byref(a), _vp(ws), ws.numel(), _stream(x)), "sf_hip_self_attention_fwd")
  return out.view(x.shape)


def transition_module(x: torch.Tensor, cond, w: dict, *, add_residual: bool = True, pre=None) -> torch.Tensor:
  """A transition block as one call (sf_hip_transition_fwd).  ``x`` ``[..., N, C]`` (leading dims =
  samples sharing the condition), ``cond`` ``[N, Cs]`` or None; ``w`` holds the packed weights
  (``w1`` ``[2I, C]`` interleaved, ``w2`` ``[C, I]``, LayerNorm / AdaLN / zero-gate terms as in
  the C struct).  ``pre`` = (scale, shift, zgate) ``[N, C]`` views with one row stride."""
  _require_cuda(x, cond, *(pre or ()))
  N, Cn = x.shape[-2], x.shape[-1]
  S = x.numel() // max(N * Cn, 1)
  w1, w2 = w["w1"], w["w2"]
  I = w2.shape[1]
  _require(tuple(w1.shape) == (2 * I, Cn) and tuple(w2.shape) == (Cn, I), "transition: weight shapes")
  x3 = _bf16(x).reshape(S, N, Cn).contiguous()
  out = torch.empty_like(x3)
  a = _lib.TransitionArgs()
  a.S, a.N, a.C, a.I = S, N, Cn, I
  a.add_residual = int(bool(add_residual))
  a.x, a.out = _vp(x3), _vp(out)
  c2 = None
  if cond is not None and pre is None:
    c2 = _bf16(cond).contiguous()
    _require(tuple(c2.shape[:-1]) == (N,), "transition: cond must be [N, Cs]")
    a.cond, a.Cs = _vp(c2), c2.shape[-1]
  for key in ("ln_w", "ln_b", "lnc_w", "lnc_b", "w_scale", "b_scale", "w_shift", "w1", "w2", "w_zc", "b_zc"):
    setattr(a, key, _vp(w.get(key)))
  if pre is not None:
    ps, pb, pz = pre
    rs = ps.stride(0)
    for t in pre:
      _require(t.dtype == torch.bfloat16 and tuple(t.shape) == (N, Cn) and t.stride() == (rs, 1),
               "transition: precomputed conditioning must be bf16 [N, C] views with one row stride")
    a.pre_scale, a.pre_shift, a.pre_zgate, a.pre_rs = _vp(ps), _vp(pb), _vp(pz), rs
  lib = _lib.load()
  nbytes = int(lib.sf_hip_transition_workspace_bytes(C.byref(a)))
  ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
  _lib.check(lib.sf_hip_transition_fwd(C.byref(a), _vp(ws), nbytes, _stream(x)), "sf_hip_transition_fwd")
  return out.view(x.shape)


def cross_attention_module(xq: torch.Tensor, xk, gather_idx, gather_mask, mask_q, mask_k, bias, cond_q, cond_k,
                           w: dict, *, num_head: int, head_dim: int, add_residual: bool = True,
                           pre: dict | None = None) -> torch.Tensor:
  """CrossAttention.forward as one call.  ``xq`` ``[..., U, Qw, C]``; keys either ``xk``
  ``[..., U, Kw, C]`` or gathered from the query rows by ``gather_idx`` / ``gather_mask``
  ``[U, Kw]``; masks ``[U, Qw]`` / ``[U, Kw]``; ``bias`` ``[U, H, Qw, Kw]``; conditions
  ``[U, Qw, C]`` / ``[U, Kw, C]``.  ``pre`` (with ``gather_idx``): the per-atom plan -- the
  keys' condition is the gathered queries', and ``pre`` holds both sides' AdaLN terms per atom
  (``q_scale``, ``q_shift``, ``k_scale``, ``k_shift``, ``zgate``: ``[U*Qw, C]`` views with one
  row stride, as cross_conditioning returns them); the conditions are then not read."""
  _require_cuda(xq, xk, gather_idx, gather_mask, mask_q, mask_k, bias, cond_q, cond_k,
                *([] if pre is None else pre.values()))
  _require(pre is None or gather_idx is not None, "cross_attention: the per-atom plan gathers its keys")
  U, Qw, Cn = xq.shape[-3:]
  S = xq.numel() // max(U * Qw * Cn, 1)
  Kw = gather_idx.shape[-1] if gather_idx is not None else xk.shape[-2]
  xq4 = _bf16(xq).reshape(S, U, Qw, Cn).contiguous()
  out = torch.empty_like(xq4)
  a = _lib.CrossAttentionArgs()
  a.S, a.U, a.Qw, a.Kw, a.C, a.H, a.D = S, U, Qw, Kw, Cn, num_head, head_dim
  a.scale, a.add_residual = 0.0, int(bool(add_residual))
  a.xq, a.out = _vp(xq4), _vp(out)
  keep = []
  if gather_idx is not None:
    idx32 = gather_idx.reshape(-1).to(torch.int32).contiguous()
    gm8 = _u8(gather_mask.reshape(-1)).contiguous()
    _require(idx32.numel() == U * Kw and gm8.numel() == U * Kw, "cross_attention: gather sizes")
    a.gather_idx, a.gather_mask = _vp(idx32), _vp(gm8)
    keep += [idx32, gm8]
  else:
    xk4 = _bf16(xk).reshape(S, U, Kw, Cn).contiguous()
    a.xk = _vp(xk4)
    keep.append(xk4)
  mq8, mk8 = _u8_or_none(mask_q), _u8_or_none(mask_k)
  a.mask_q, a.mask_k = _vp(mq8), _vp(mk8)
  b = None if bias is None else _bf16(bias).contiguous()
  a.bias = _vp(b)
  if pre is None:
    cq, ck = _bf16(cond_q).contiguous(), _bf16(cond_k).contiguous()
    a.cond_q, a.cond_k = _vp(cq), _vp(ck)
  else:
    terms = [pre[k] for k in ("q_scale", "q_shift", "k_scale", "k_shift", "zgate")]
    rs = terms[0].stride(0)
    for t in terms:
      _require(t.dtype == torch.bfloat16 and tuple(t.shape) == (U * Qw, Cn) and t.stride() == (rs, 1),
               "cross_attention: pre terms must be bf16 [U*Qw, C] views with one row stride")
    a.pre_q_scale, a.pre_q_shift, a.pre_k_scale, a.pre_k_shift, a.pre_zgate = (_vp(t) for t in terms)
    a.pre_rs = rs
  for key in ("lnc_w_q", "lnc_b_q", "w_scale_q", "b_scale_q", "w_shift_q", "lnc_w_k", "lnc_b_k", "w_scale_k",
              "b_scale_k", "w_shift_k", "w_qg", "b_qg", "w_kv", "w_t2", "w_zc", "b_zc"):
    setattr(a, key, _vp(w.get(key)))
  lib = _lib.load()
  ws = torch.empty(int(lib.sf_hip_cross_attention_workspace_bytes(C.byref(a))), dtype=torch.uint8, device=xq.device)
  _lib.check(lib.sf_hip_cross_attention_fwd(C.byref(a), _vp(ws), ws.numel(), _stream(xq)), "sf_hip_cross_attention_fwd")
  return out.view(xq.shape)


def diffusion_conditioning(cond: torch.Tensor, lnc_w: torch.Tensor, w_scale: torch.Tensor, b_scale, w_shift: torch.Tensor,
                           w_zc: torch.Tensor, b_zc) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
  """AdaLN conditioning of L layers from one condition, one call (sf_hip_diffusion_conditioning_fwd;
  the reference's diffusion_conditioning_packed, backends/vecops/kernels/registry.py:720-760).
  ``cond`` ``[..., N, Cs]``; ``lnc_w`` f32 ``[L, Cs]``; weights bf16 ``[L*C, Cs]``; biases f32
  ``[L*C]``.  Returns (scale, shift, zgate), each ``[L, rows, C]`` (rows = cond's leading dims x N)
  as per-layer views of one ``[rows, L*C]`` buffer; scale and zgate after the sigmoid."""
  _require_cuda(cond, lnc_w, w_scale, b_scale, w_shift, w_zc, b_zc)
  L, Cs = lnc_w.shape
  LC = w_scale.shape[0]
  _require(LC % L == 0 and cond.shape[-1] == Cs, "diffusion_conditioning: shapes do not match")
  Cn = LC // L
  for t, n in ((w_scale, "w_scale"), (w_shift, "w_shift"), (w_zc, "w_zc")):
    _require(tuple(t.shape) == (LC, Cs) and t.dtype == torch.bfloat16 and t.is_contiguous(),
             f"diffusion_conditioning: {n} must be contiguous bf16 [L*C, Cs]")
  c2 = _bf16(cond).reshape(-1, Cs).contiguous()
  rows = c2.shape[0]
  outs = [torch.empty(rows, LC, dtype=torch.bfloat16, device=cond.device) for _ in range(3)]
  a = _lib.DiffusionConditioningArgs()
  a.rows, a.L, a.C, a.Cs = rows, L, Cn, Cs
  g = lnc_w.float().contiguous()
  bs = None if b_scale is None else b_scale.float().contiguous()
  bz = None if b_zc is None else b_zc.float().contiguous()
  a.cond, a.lnc_w, a.w_scale, a.b_scale, a.w_shift = _vp(c2), _vp(g), _vp(w_scale), _vp(bs), _vp(w_shift)
  a.w_zc, a.b_zc = _vp(w_zc), _vp(bz)
  a.scale, a.shift, a.zgate, a.out_rs = _vp(outs[0]), _vp(outs[1]), _vp(outs[2]), LC
  lib = _lib.load()
  ws = torch.empty(int(lib.sf_hip_diffusion_conditioning_workspace_bytes(C.byref(a))), dtype=torch.uint8,
                   device=cond.device)
  _lib.check(lib.sf_hip_diffusion_conditioning_fwd(C.byref(a), _vp(ws), ws.numel(), _stream(cond)),
             "sf_hip_diffusion_conditioning_fwd")
  return tuple(o.view(rows, L, Cn).transpose(0, 1) for o in outs)


def triangle_multiplication(z: torch.Tensor, mask, w: dict, *, incoming: bool, add_residual: bool = True) -> torch.Tensor:
  """TriangleMultiplication.forward (blocks.py:486-566) as one call (sf_hip_triangle_mult_fwd).
  ``z`` ``[N, N, 128]``, ``mask`` ``[N]`` bool or None; ``w`` holds the packed weights (keys as in
  the C struct)."""
  _require_cuda(z, mask)
  _require(z.dim() == 3 and z.shape[0] == z.shape[1], "triangle_multiplication: z must be [N, N, C]")
  N, Cn = z.shape[0], z.shape[2]
  z3 = _bf16(z).contiguous()
  out = torch.empty_like(z3)
  lib = _lib.load()
  ws_bytes = int(lib.sf_hip_triangle_mult_workspace_bytes(N, Cn))
  if ws_bytes <= 0:
    raise ValueError(f"triangle_multiplication: unsupported sizes N={N} C={Cn} (C must be 128)")
  a = _lib.TriangleMultArgs()
  a.N, a.C, a.incoming, a.add_residual = N, Cn, int(bool(incoming)), int(bool(add_residual))
  m8 = _u8_or_none(mask)
  a.z, a.mask, a.out = _vp(z3), _vp(m8), _vp(out)
  for key in ("ln_w", "ln_b", "w_glu", "cn_w", "cn_b", "w_out", "w_gate"):
    setattr(a, key, _vp(w.get(key)))
  ws = torch.empty(ws_bytes, dtype=torch.uint8, device=z.device)
  _lib.check(lib.sf_hip_triangle_mult_fwd(C.byref(a), _vp(ws), ws.numel(), _stream(z)), "sf_hip_triangle_mult_fwd")
  return out.to(z.dtype) if z.dtype != torch.bfloat16 else out


# ---------------------------------------------------------------------------------------
# packed sequences: attention, rotary positions, norm of queries and keys with the rotation
# (sf_hip_packed_attention_fwd, sf_hip_rotary_fwd)
# ---------------------------------------------------------------------------------------

_ELEMENT_TYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_NORMS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}


def _no_grad(what: str, *ts) -> None:
  """These calls have no backward pass and no tangents: a tensor that expects a gradient or carries a tangent through them
  is refused."""
  if torch.is_grad_enabled():
    for t in ts:
      if t is not None and t.requires_grad:
        raise ValueError(f"{what}: has no backward pass; detach the inputs or call it under torch.no_grad()")
  if forward_ad._current_level >= 0:                           # (inside a dual level)
    for t in ts:
      if t is not None and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what}: has no forward-mode derivative; pass the primals of dual tensors")


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(fn, t: torch.Tensor, what: str, *args) -> None:
  """``fn(*args, stream)`` with t's device current."""
  index = t.get_device()
  if index == _current_device():
    _lib.check(fn(*args, _stream(t)), what)
  else:
    with torch.cuda.device(index):
      _lib.check(fn(*args, _stream(t)), what)


def _fresh(t: torch.Tensor) -> torch.Tensor:
  """An uninitialised packed tensor like t (half the host time of ``torch.empty`` with a shape)."""
  return torch.empty_like(t, memory_format=torch.contiguous_format)


def _strides2(t: torch.Tensor) -> tuple[int, int]:
  """Row and head strides of ``[T, H, D]``; those of a single row or head, which torch leaves
  arbitrary, as if packed."""
  T, H, D = t.shape
  st, sh, _ = t.stride()
  if H <= 1:
    sh = D
  return (st if T > 1 else max(H * sh, H * D)), sh


def _extent(t: torch.Tensor) -> tuple[int, int, int]:
  """First byte, row stride and bytes of one row of ``[T, H, D]``."""
  st, sh = _strides2(t)
  return t.data_ptr(), st * t.element_size(), ((t.shape[1] - 1) * sh + t.shape[2]) * t.element_size()


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
  """Whether two ``[T, H, D]`` views share no element: separate ranges, or separate columns of rows
  of one width."""
  if a.numel() == 0 or b.numel() == 0:
    return True
  (pa, sa, ea), (pb, sb, eb) = _extent(a), _extent(b)
  if pa + (a.shape[0] - 1) * sa + ea <= pb or pb + (b.shape[0] - 1) * sb + eb <= pa:
    return True
  return sa == sb and ea <= sa and eb <= sa and eb <= (pa - pb) % sa <= sa - ea


def _separate(t: torch.Tensor) -> bool:
  """Whether the rows and heads of a ``[T, H, D]`` view lie apart, row-major or head-major."""
  st, sh = _strides2(t)
  T, H, D = t.shape
  return t.numel() == 0 or (sh >= D and st >= (H - 1) * sh + D) or (st >= D and sh >= (T - 1) * st + D)


_increment_version = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


def _written(*ts) -> None:
  """Tells autograd that the caller's tensors were written: a graph that saved their old values refuses to use them."""
  for t in ts:
    if t is not None and not t.is_inference():
      _increment_version((t,))


def _offsets32(t: torch.Tensor, name: str, n: int | None, what: str) -> torch.Tensor:
  if t.dtype is not torch.int32 or t.ndim != 1 or (n is not None and t.shape[0] != n):
    raise ValueError(f"{what}: {name} must be int32 [{'sequences + 1' if n is None else n}], got {t.dtype} {tuple(t.shape)}")
  return t if t.is_contiguous() else t.contiguous()


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor | None = None, *, len_q: torch.Tensor | None = None,
                     len_k: torch.Tensor | None = None, causal: bool = False, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
  """Attention over packed sequences of different lengths; returns ``out`` like ``q``.

  ``q`` ``[Tq, H, D]``, ``k`` and ``v`` ``[Tk, Hkv, D]``, bf16 or fp16 (one type), ``H`` a multiple of
  ``Hkv``: query head h reads key head ``h // (H // Hkv)``.  ``D`` a multiple of 8 up to 128.  Any row
  and head strides (columns of a fused projection, a cache); what is not in 16-byte aligned rows is
  copied first.

  ``cu_q`` int32 ``[B + 1]`` on the device: sequence b has the query rows ``cu_q[b] .. cu_q[b+1] - 1``;
  ``cu_k`` the same for its keys (None: the queries' offsets, and their ``len_q``).  ``len_q`` /
  ``len_k`` int32 ``[B]``: only that many rows of each are in use (a padded batch, a cache with free
  rows).  With ``causal``, query i of n sees keys ``j <= i + m - n`` of m: the last query sees all, so a
  new token or the rest of a prompt attends to a cache.  A query without a key gives zeros.  Rows
  of ``out`` outside every sequence are left as they were: undefined unless ``out`` is given.

  The offsets are read on the device only: the call neither synchronises nor copies them, and can
  be captured.  They must not decrease; wrong ones give wrong results but no access outside the
  tensors.  ``out`` may not overlap an input."""
  what = "packed_attention"
  _no_grad(what, q, k, v, out)
  dev = _require_cuda(q, k, v, cu_q, cu_k, len_q, len_k, out)
  qs, ks = q.shape, k.shape
  _require(len(qs) == 3 and len(ks) == 3 and v.ndim == 3, "packed_attention: q, k and v must be [tokens, heads, dim]")
  Tq, H, D = qs
  Tk, Hkv, Dk = ks
  if Dk != D or v.shape != ks:
    raise ValueError(f"packed_attention: shapes q{tuple(qs)} k{tuple(ks)} v{tuple(v.shape)}")
  if H == 0 or Hkv == 0 or H % Hkv != 0 or H > 1 << 24:
    raise ValueError(f"packed_attention: {H} query heads do not share {Hkv} key heads evenly, or exceed 2^24")
  if D % 8 != 0 or not 0 < D <= 128:
    raise ValueError(f"packed_attention: head dim {D} is not a multiple of 8 up to 128")
  dtype = q.dtype
  if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype is not dtype or v.dtype is not dtype:
    raise ValueError(f"packed_attention: q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}")
  cu_q = _offsets32(cu_q, "cu_q", None, what)
  B = cu_q.shape[0] - 1
  _require(1 <= B < 1 << 30, "packed_attention: cu_q needs at least two offsets, and below 2^30")
  if cu_k is None:
    cu_k, len_k = cu_q, (len_q if len_k is None else len_k)
  else:
    cu_k = _offsets32(cu_k, "cu_k", B + 1, what)
  if len_q is not None:
    len_q = _offsets32(len_q, "len_q", B, what)
  if len_k is not None:
    len_k = _offsets32(len_k, "len_k", B, what)
  scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
  if not abs(scale) <= 1e30:
    raise ValueError(f"packed_attention: scale {scale} is not finite or above 1e30")

  def rows(t, least):
    ptr = t.data_ptr()
    if t.is_contiguous() and ptr % 16 == 0 and t.shape[1] * D < 1 << 24:
      return t, ptr, (t.shape[1] * D, D)
    st, sh, sd = t.stride()
    if t.shape[1] == 1:                                        # (a single head's or row's stride means nothing)
      sh = D
    if t.shape[0] <= 1:
      st = t.shape[1] * max(sh, D)
    if sd != 1 or (st | sh | ptr >> 1) % 8 or not least <= st < 1 << 24:
      t = torch.empty(t.shape, dtype=dtype, device=dev).copy_(t)
      st, sh, ptr = t.shape[1] * D, D, t.data_ptr()
    return t, ptr, (st, sh)

  given = out
  if out is None:
    out = _fresh(q)
    so = (H * D, D)
  else:
    so = _strides2(out) if out.ndim == 3 else (0, 0)
    if (out.shape != qs or out.dtype != dtype or out.stride(2) != 1 or so[0] % 8 or so[1] % 8 or out.data_ptr() % 16
        or not _separate(out)):
      raise ValueError(f"packed_attention: out must be {dtype} {(Tq, H, D)} in 16-byte aligned rows, apart from each other")
    if not (_disjoint(out, q) and _disjoint(out, k) and _disjoint(out, v)):
      raise ValueError("packed_attention: out overlaps an input")
  q, qp, sq = rows(q, 0)
  k, kp, sk = rows(k, D)
  v, vp, sv = rows(v, D)
  a = _lib.packed_attention_args(B, H, Hkv, D, Tq, Tk, scale, bool(causal), _ELEMENT_TYPES[dtype], qp, *sq, kp, *sk, vp, *sv,
                                 out.data_ptr(), *so, cu_q.data_ptr(), cu_k.data_ptr(), _vp(len_q) or 0, _vp(len_k) or 0)
  lib = _lib.load()
  ref = C.byref(a)
  need = lib.sf_hip_packed_attention_workspace_bytes(ref)
  ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
  _launch(lib.sf_hip_packed_attention_fwd, q, "sf_hip_packed_attention_fwd", ref, _vp(ws), need)
  _written(given)
  return out


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> torch.Tensor:
  """Radians per position of the ``rotary_dim / 2`` pairs, float64: ``base ** (-2 i / rotary_dim)``,
  stretched for contexts ``factor`` times longer than the trained ones where ``scaling`` says how:

  * ``"linear"``  every frequency divided by ``factor`` (positions interpolated);
  * ``"base"``    ``base`` raised so that the slowest pair is divided by ``factor`` and the fastest stays;
  * ``"turns"``   by the turns that a pair makes over ``original_length`` positions: from
    ``high_turns`` on it stays, up to ``low_turns`` it is divided by ``factor``, between them linearly blended.

  A set-up step on the host; a program keeps the tensor."""
  _require(rotary_dim >= 2 and rotary_dim % 2 == 0, f"rotary_frequencies: rotary_dim {rotary_dim} is not even and positive")
  _require(base > 0 and factor > 0, "rotary_frequencies: base and factor must be positive")
  exponents = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
  if scaling == "base":
    _require(rotary_dim > 2, "rotary_frequencies: scaling 'base' needs at least two pairs")
    base = base * factor ** (rotary_dim / (rotary_dim - 2))
  freqs = float(base) ** -exponents
  if scaling == "linear":
    freqs = freqs / factor
  elif scaling == "turns":
    _require(original_length is not None and original_length > 0 and high_turns > low_turns,
             "rotary_frequencies: scaling 'turns' needs original_length > 0 and high_turns > low_turns")
    keep = ((original_length * freqs / (2.0 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
    freqs = freqs * (keep + (1.0 - keep) / factor)
  else:
    _require(scaling in (None, "base"), f"rotary_frequencies: scaling {scaling!r} is not None, 'linear', 'base' or 'turns'")
  return freqs.to(device) if device is not None else freqs


def _rotary(what, q, k, positions, freqs, interleaved, magnitude, out_q, out_k, norm=0, eps=0.0, weights=(None,) * 4):
  _no_grad(what, q, k, freqs, out_q, out_k, *weights)
  _require_cuda(q, k, positions, freqs, out_q, out_k, *weights)
  qs, ks = q.shape, None if k is None else k.shape
  nd = len(qs)
  if nd < 3 or (ks is not None and (len(ks) != nd or ks[-1] != qs[-1] or (ks[0] != qs[0] if nd == 3 else ks[:-2] != qs[:-2]))):
    raise ValueError(f"{what}: q must be [..., H, D] and k [..., Hk, D], got {tuple(qs)}{'' if ks is None else ' and ' + str(tuple(ks))}")
  H, D = qs[-2], qs[-1]
  dtype = q.dtype
  if dtype not in _ELEMENT_TYPES or (k is not None and k.dtype != dtype):
    raise ValueError(f"{what}: q and k must be bfloat16, float16 or float32 alike, got {dtype}{'' if k is None else f' and {k.dtype}'}")
  if not 0 < H <= 1 << 24 or (ks is not None and not 0 < ks[-2] <= 1 << 24) or not 0 < D <= 256:
    raise ValueError(f"{what}: heads must lie in 1 .. 2^24 and head dims lie in 1 .. 256, got {tuple(q.shape)}")
  pairs = freqs.numel()
  if freqs.dtype != torch.float64 or freqs.ndim != 1 or not 1 <= pairs <= D // 2:
    raise ValueError(f"{what}: freqs must be float64 [R / 2], 1 to {D // 2} of them, got {freqs.dtype} {tuple(freqs.shape)}")
  pdtype = positions.dtype
  if pdtype is not torch.int32 and pdtype is not torch.int64:
    raise ValueError(f"{what}: positions must be int32 or int64, got {pdtype}")
  flat = nd == 3
  if positions.ndim != 1 or not flat or positions.shape[0] != qs[0]:
    try:
      positions = positions.expand(qs[:-2])
    except RuntimeError:
      raise ValueError(f"{what}: positions {tuple(positions.shape)} do not fit tokens {tuple(qs[:-2])}") from None
    positions = positions.reshape(-1)
  if not abs(magnitude) <= 1e30:
    raise ValueError(f"{what}: magnitude {magnitude} is not finite or above 1e30")

  def three(t):
    t3 = t if flat else t.reshape(-1, t.shape[-2], D)
    t3 = t3 if t3.stride(2) == 1 else t3.contiguous()
    return t3, _strides2(t3)

  def given(o, like, name):
    if o.shape != like.shape or o.dtype != dtype or (D > 1 and o.stride(-1) != 1):
      raise ValueError(f"{what}: {name} must be {dtype} {tuple(like.shape)} with a unit last stride")
    try:
      o = o if flat else o.view(-1, o.shape[-2], D)
    except RuntimeError:
      raise ValueError(f"{what}: the leading dims of {name} must be one stride apart") from None
    if not _separate(o):
      raise ValueError(f"{what}: {name} must hold every element once")
    return o

  if k is None and out_k is not None:
    raise ValueError(f"{what}: out_k without k")
  given_q, given_k = out_q, out_k
  q3, sq = (q, (H * D, D)) if flat and q.is_contiguous() else three(q)
  T = q3.shape[0]
  if out_q is None:
    out_q = _fresh(q)
    oq3, so = out_q, (H * D, D)
  else:
    oq3 = given(out_q, q, "out_q")
    so = _strides2(oq3)
  Hk, k3, ok3, kp, sk, okp, sok = 0, None, None, 0, (0, 0), 0, (0, 0)
  if k is not None:
    Hk = ks[-2]
    k3, sk = (k, (Hk * D, D)) if flat and k.is_contiguous() else three(k)
    kp = k3.data_ptr()
    if out_k is None:
      out_k = _fresh(k)
      ok3, sok = out_k, (Hk * D, D)
    else:
      ok3 = given(out_k, k, "out_k")
      sok = _strides2(ok3)
    okp = ok3.data_ptr()
  if given_q is not None or given_k is not None:
    same = lambda a, b: a.data_ptr() == b.data_ptr() and a.shape == b.shape and _strides2(a) == _strides2(b)
    oq, ok = oq3.view(-1, H, D) if oq3.ndim != 3 else oq3, ok3.view(-1, Hk, D) if ok3 is not None and ok3.ndim != 3 else ok3
    meets = [(oq, q3, True)] if k is None else [(oq, q3, True), (ok, k3, True), (oq, k3, False), (ok, q3, False), (oq, ok, False)]
    for a, b, own in meets:
      if not (_disjoint(a, b) or (own and same(a, b))):
        raise ValueError(f"{what}: outputs may be their own input in place, and overlap nothing else")
  if not positions.is_contiguous():
    positions = positions.contiguous()
  if not freqs.is_contiguous():
    freqs = freqs.contiguous()
  qw, kw, qb, kb = weights
  a = _lib.rotary_args(T, H, Hk, D, 2 * pairs, bool(interleaved), _ELEMENT_TYPES[dtype], norm, eps, magnitude, q3.data_ptr(), *sq,
                       kp, *sk, oq3.data_ptr(), *so, okp, *sok, positions.data_ptr(), pdtype is torch.int64, freqs.data_ptr(),
                       _vp(qw) or 0, _vp(qb) or 0, _vp(kw) or 0, _vp(kb) or 0)
  _launch(_lib.load().sf_hip_rotary_fwd, q3, "sf_hip_rotary_fwd", C.byref(a))
  _written(given_q, given_k)
  return out_q, out_k


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
           interleaved: bool = False, magnitude: float = 1.0, out_q: torch.Tensor | None = None,
           out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
  """Rotary positions of ``q`` ``[..., H, D]`` and ``k`` ``[..., Hk, D]`` (or None); returns both turned.

  The first ``R = 2 * len(freqs)`` dims of each head are turned in pairs, ``(i, i + R/2)`` or with
  ``interleaved`` ``(2i, 2i + 1)``, by ``positions * freqs[i]`` radians and multiplied by ``magnitude``; the
  others are copied.  ``positions`` int32 or int64 of the tokens' leading dims (broadcast where they are
  fewer), ``freqs`` float64 on the device (``rotary_frequencies``).  bf16, fp16 or float32, head dims up
  to 256, any strides with a unit last one.  The angle is formed in 64 bits, the rest in 32, rounded
  once.  ``out_q`` may be ``q`` and ``out_k`` may be ``k`` (in place); they overlap nothing else."""
  return _rotary("rotary", q, k, positions, freqs, interleaved, magnitude, out_q, out_k)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                   positions: torch.Tensor, freqs: torch.Tensor, *, norm: str = "rms", eps: float = 1e-6,
                   q_bias: torch.Tensor | None = None, k_bias: torch.Tensor | None = None, interleaved: bool = False,
                   magnitude: float = 1.0, out_q: torch.Tensor | None = None,
                   out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
  """Norm of each query and key head, then their rotary positions, in one pass; arguments and results
  as ``rotary``.  ``norm`` ``"rms"``: ``x rsqrt(mean x^2 + eps) weight``; ``"layer"``:
  ``(x - mean) rsqrt(var + eps) weight + bias``, over the D dims of a head.  Weights and biases ``[D]``
  (None: 1 and 0; biases with ``"layer"`` only), float32; others are cast at every call."""
  what = "qk_norm_rotary"
  if norm not in _NORMS:
    raise ValueError(f"{what}: norm {norm!r} is not 'rms' or 'layer'")
  if norm == "rms" and (q_bias is not None or k_bias is not None):
    raise ValueError(f"{what}: biases need norm='layer'")
  if k is None and (k_weight is not None or k_bias is not None):
    raise ValueError(f"{what}: a key weight or bias without k")
  if not 0.0 <= eps <= 1e30:
    raise ValueError(f"{what}: eps {eps} is not finite and >= 0, or above 1e30")
  weights, D = (q_weight, k_weight, q_bias, k_bias), q.shape[-1]
  for w in weights:
    if w is not None:
      if w.shape != (D,):
        raise ValueError(f"{what}: weights and biases must be [{D}], got {tuple(w.shape)}")
      if w.dtype is not torch.float32 or not w.is_contiguous():
        _no_grad(what, *weights)
        weights = tuple(x if x is None else _f32(x) for x in weights)
  return _rotary(what, q, k, positions, freqs, interleaved, magnitude, out_q, out_k, _NORMS[norm], float(eps), weights)


# ---------------------------------------------------------------------------------------
# a paged cache of keys and values: new rows into their pages, attention over them
# (sf_hip_paged_write_fwd, sf_hip_paged_attention_fwd)
# ---------------------------------------------------------------------------------------

_front = None


def _library():
  """The library, for the calls from here on; with it their host module is loaded, which takes their common form from then on
  (a norm of 8 rows 9.9 -> 5.7 us of host time, a cache write of 64 tokens 10.8 -> 4.0)."""
  global _front
  lib = _lib.load()
  if _front is None:
    _front = _lib.front(lib, Microscaled) or False
  return lib


def _page_strides(t: torch.Tensor) -> tuple[int, int, int]:
  """Page, row and head strides of ``[pages, rows, heads, D]``; those of a single page or head, which torch leaves
  arbitrary, as if packed."""
  P, R, H, D = t.shape
  sp, sr, sh, _ = t.stride()
  if H == 1:
    sh = D
  return (sp if P > 1 else max(R * sr, H * sh)), sr, sh


def _apart(dims) -> bool:
  """Whether a view holds every element once, by (size, stride) of its dims: each lies outside what the narrower ones span."""
  reach = 1
  for size, stride in sorted((d for d in dims if d[0] > 1), key=lambda d: d[1]):
    if stride < reach:
      return False
    reach += (size - 1) * stride
  return True


def _span(t: torch.Tensor) -> tuple[int, int]:
  """First byte and the byte past the last of a view with non-negative strides."""
  p, n = t.data_ptr(), t.numel()
  if n > 0 and not t.is_contiguous():
    n = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
  return p, p + n * t.element_size()


def _spans_apart(a: torch.Tensor, b: torch.Tensor) -> bool:
  (a0, a1), (b0, b1) = _span(a), _span(b)
  return a1 <= b0 or b1 <= a0 or a0 == a1 or b0 == b1


def _cache(what, k_pages, v_pages, page_table, len_k, B, dtype):
  """Checks a paged cache; returns its strides, the table's pointer, row stride and width, and the table and lengths kept alive."""
  shape = k_pages.shape
  if len(shape) != 4 or v_pages.shape != shape or k_pages.dtype is not dtype or v_pages.dtype is not dtype:
    raise ValueError(f"{what}: k_pages and v_pages must be {dtype} [pages, rows, heads, dim] alike, got {k_pages.dtype} {tuple(shape)} "
                     f"and {v_pages.dtype} {tuple(v_pages.shape)}")
  P, R, Hkv, D = shape
  if P < 1 or R < 16 or R % 16 or Hkv < 1:
    raise ValueError(f"{what}: a cache needs pages of a multiple of 16 rows, got {tuple(shape)}")
  if D % 8 != 0 or not 0 < D <= 128:
    raise ValueError(f"{what}: head dim {D} is not a multiple of 8 up to 128")
  row = Hkv * D
  packed = (R * row, row, D)
  strides = []
  for t in (k_pages, v_pages):
    whole = t.is_contiguous()
    s = packed if whole else _page_strides(t)
    if t.data_ptr() % 16 or not (row < 1 << 24 if whole else not (s[0] | s[1] | s[2]) % 8 and D <= s[1] < 1 << 24 and t.stride(3) == 1):
      raise ValueError(f"{what}: pages must lie in 16-byte aligned rows of 1 dim after another, strides {t.stride()}")
    strides.append(s)
  tshape = page_table.shape
  cols = tshape[1] if len(tshape) == 2 else 0
  if page_table.dtype is not torch.int32 or cols < 1 or tshape[0] != B:
    raise ValueError(f"{what}: page_table must be int32 [{B}, pages of a sequence], got {page_table.dtype} {tuple(tshape)}")
  if cols * R > 1 << 30:
    raise ValueError(f"{what}: {cols} pages of {R} rows a sequence exceed 2^30")
  ts = cols
  if not page_table.is_contiguous():
    if cols > 1 and page_table.stride(1) != 1:
      page_table = page_table.contiguous()
    elif B > 1:
      ts = page_table.stride(0)
  return *strides, page_table, ts, cols, _offsets32(len_k, "len_k", B, what)


def _token_rows(t: torch.Tensor, T: int, H: int, D: int):
  """``[T, H, D]`` in 16-byte aligned rows (copied where it is not): the tensor, its pointer and strides."""
  ptr = t.data_ptr()
  if ptr % 16 == 0 and t.is_contiguous():
    return t, ptr, (H * D, D)
  st, sh, sd = t.stride()
  if sd == 1 and T > 1 and H > 1 and not (st | sh | ptr >> 1) % 8:
    return t, ptr, (st, sh)
  st, sh = _strides2(t)
  if t.stride(2) != 1 or (st | sh | ptr >> 1) % 8:
    t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    (st, sh), ptr = (H * D, D), t.data_ptr()
  return t, ptr, (st, sh)


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                      cu: torch.Tensor, len_k: torch.Tensor, *, len_new: torch.Tensor | None = None) -> None:
  """Writes new keys and values into their pages.

  ``k`` and ``v`` ``[T, Hkv, D]``: sequence b's new tokens are rows ``cu[b] .. cu[b+1] - 1`` (``cu`` int32 ``[B + 1]``; with
  ``len_new`` int32 ``[B]`` only the first that many).  ``len_k`` int32 ``[B]`` counts a sequence's keys with the new ones:
  of n new rows, row i becomes its key ``len_k[b] - n + i``.  ``k_pages`` and ``v_pages`` ``[pages, rows, Hkv, D]`` of the same
  type, bf16 or fp16, pages of a multiple of 16 rows, any strides of 16-byte aligned rows; key j of sequence b lies in row
  ``j % rows`` of page ``page_table[b, j // rows]`` (int32 ``[B, pages of a sequence]``).

  Offsets, lengths and table are read on the device only: the call can be captured.  Keys whose place lies outside the
  table or the cache are dropped.  Each new key has a place of its own: pages that sequences share are written by one of
  them at most, and a sequence's table names a page once (of two keys written to one place either is left)."""
  if _front and _front.paged_cache_write(k, v, k_pages, v_pages, page_table, cu, len_k, len_new):
    return
  what = "paged_cache_write"
  _no_grad(what, k, v, k_pages, v_pages)
  _require_cuda(k, v, k_pages, v_pages, page_table, cu, len_k, len_new)
  dtype = k.dtype
  if k.ndim != 3 or v.shape != k.shape or v.dtype is not dtype or (dtype is not torch.bfloat16 and dtype is not torch.float16):
    raise ValueError(f"{what}: k and v must be [tokens, heads, dim], both bfloat16 or float16, got {k.dtype} {tuple(k.shape)} and "
                     f"{v.dtype} {tuple(v.shape)}")
  T, Hkv, D = k.shape
  cu = _offsets32(cu, "cu", None, what)
  B = cu.shape[0] - 1
  _require(1 <= B < 1 << 30 and T <= 1 << 30, "paged_cache_write: cu needs at least two offsets, up to 2^30 tokens")
  if len_new is not None:
    len_new = _offsets32(len_new, "len_new", B, what)
  ks, vs, table, ts, cols, len_k = _cache(what, k_pages, v_pages, page_table, len_k, B, dtype)
  P, R, Hp, Dp = k_pages.shape
  if Hp != Hkv or Dp != D or Hkv * D > 1 << 24:
    raise ValueError(f"{what}: {tuple(k.shape[1:])} of k and v against {tuple(k_pages.shape[2:])} of the pages (2^24 elements at most)")
  packed = (R * Hkv * D, Hkv * D, D)
  for pages, strides in ((k_pages, ks), (v_pages, vs)):
    if strides != packed and not _apart(zip(pages.shape, (*strides, 1))):
      raise ValueError(f"{what}: pages must hold every element once")
  k0, v0 = k_pages.data_ptr(), v_pages.data_ptr()
  k1, v1 = (p + 2 * ((P - 1) * s[0] + (R - 1) * s[1] + (Hkv - 1) * s[2] + D) for p, s in ((k0, ks), (v0, vs)))
  if not (k1 <= v0 or v1 <= k0 or (ks == vs and _apart([*zip(k_pages.shape, (*ks, 1)), (2, abs(v0 - k0) // 2)]))):
    raise ValueError(f"{what}: k_pages and v_pages overlap")
  k, kp, sk = _token_rows(k, T, Hkv, D)                        # (copies overlap nothing)
  v, vp, sv = _token_rows(v, T, Hkv, D)
  for p, (st, sh) in ((kp, sk), (vp, sv)):
    end = p + 2 * ((T - 1) * st + (Hkv - 1) * sh + D)
    if T > 0 and not ((end <= k0 or k1 <= p) and (end <= v0 or v1 <= p)):
      raise ValueError(f"{what}: pages overlap k or v")
  a = _lib.paged_write_args(B, Hkv, D, T, P, R, cols, kp, *sk, vp, *sv, k0, *ks, v0, *vs, cu.data_ptr(), _vp(len_new) or 0,
                            len_k.data_ptr(), table.data_ptr(), ts)
  _launch(_library().sf_hip_paged_write_fwd, k, "sf_hip_paged_write_fwd", C.byref(a))
  _written(k_pages, v_pages)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cu_q: torch.Tensor,
                    len_k: torch.Tensor, *, len_q: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
                    max_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
  """Attention of new tokens over a paged cache that holds their keys already (``paged_cache_write``); returns ``out``
  like ``q``.

  ``q`` ``[Tq, H, D]``, ``cu_q``, ``len_q``, ``causal``, ``scale`` and ``out`` as in ``packed_attention``; the cache, ``page_table``
  and ``len_k`` as in ``paged_cache_write``, ``H`` a multiple of its heads.  With ``causal``, query i of n sees keys
  ``j <= i + len_k - n``: one new token a sequence, a piece of a prompt, or both in one call.  A query without a key
  gives zeros; rows of ``out`` outside every sequence are left as they were.  Sequences may share pages.

  ``max_len``: the most keys that a sequence has (None: what the table holds).  The launch is chosen by it; a wrong one costs
  time, no result.  Offsets, lengths and table are read on the device only: the call can be captured.  What pages hold behind
  a sequence's end has no influence; a page outside the cache counts as zeros.

  Logits, sums and results are fp32 up to their rounding; the weights are rounded to the type of ``q`` for the product with the values, and
  the sum takes the rounded ones, as in ``packed_attention`` (errors up to 1.4 times those of 32-bit weights)."""
  if _front and out is None:
    result = _front.paged_attention(q, k_pages, v_pages, page_table, cu_q, len_k, len_q, causal, scale, max_len)
    if result is not None:
      return result
  what = "paged_attention"
  _no_grad(what, q, k_pages, v_pages, out)
  dev = _require_cuda(q, k_pages, v_pages, page_table, cu_q, len_k, len_q, out)
  qs, dtype = q.shape, q.dtype
  if len(qs) != 3 or (dtype is not torch.bfloat16 and dtype is not torch.float16):
    raise ValueError(f"{what}: q must be bfloat16 or float16 [tokens, heads, dim], got {dtype} {tuple(qs)}")
  Tq, H, D = qs
  cu_q = _offsets32(cu_q, "cu_q", None, what)
  B = cu_q.shape[0] - 1
  _require(1 <= B < 1 << 30, "paged_attention: cu_q needs at least two offsets, and below 2^30")
  if len_q is not None:
    len_q = _offsets32(len_q, "len_q", B, what)
  ks, vs, table, ts, cols, len_k = _cache(what, k_pages, v_pages, page_table, len_k, B, dtype)
  P, R, Hkv, Dk = k_pages.shape
  if Dk != D or H == 0 or H % Hkv != 0 or H > 1 << 24:
    raise ValueError(f"{what}: q {tuple(qs)} against pages {tuple(k_pages.shape)}: one head dim, heads that share key heads evenly")
  scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
  if not abs(scale) <= 1e30:
    raise ValueError(f"{what}: scale {scale} is not finite or above 1e30")
  if max_len is not None and not 0 <= max_len < 1 << 62:
    raise ValueError(f"{what}: max_len {max_len} is negative or too large")
  given = out
  if out is None:
    out, so = _fresh(q), (H * D, D)
  else:
    so = _strides2(out) if out.ndim == 3 else (0, 0)
    if (out.shape != qs or out.dtype != dtype or out.stride(2) != 1 or so[0] % 8 or so[1] % 8 or out.data_ptr() % 16
        or not _separate(out)):
      raise ValueError(f"{what}: out must be {dtype} {(Tq, H, D)} in 16-byte aligned rows, apart from each other")
    if not (_disjoint(out, q) and _spans_apart(out, k_pages) and _spans_apart(out, v_pages)):
      raise ValueError(f"{what}: out overlaps an input")
  q, qp, sq = _token_rows(q, Tq, H, D)
  a = _lib.paged_attention_args(B, H, Hkv, D, Tq, P, R, cols, max(max_len, 1) if max_len is not None else 0, scale, bool(causal),
                                _ELEMENT_TYPES[dtype], qp, *sq, k_pages.data_ptr(), *ks, v_pages.data_ptr(), *vs, out.data_ptr(), *so,
                                cu_q.data_ptr(), _vp(len_q) or 0, len_k.data_ptr(), table.data_ptr(), ts)
  lib = _library()
  ref = C.byref(a)
  need = lib.sf_hip_paged_attention_workspace_bytes(ref)
  ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
  _launch(lib.sf_hip_paged_attention_fwd, q, "sf_hip_paged_attention_fwd", ref, _vp(ws), need)
  _written(given)
  return out


# ---------------------------------------------------------------------------------------
# microscaled numbers, their product, and the residual's addition with the norm
# (sf_hip_mx_encode_fwd, sf_hip_mx_decode_fwd, sf_hip_mx_linear_fwd, sf_hip_add_rms_norm_fwd)
# ---------------------------------------------------------------------------------------

_FORMATS = {"mxfp8": _lib.FORMAT_MXFP8, "mxfp4": _lib.FORMAT_MXFP4}
_FP8, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class Microscaled(NamedTuple):
  """Numbers in blocks of 32 along the last dim that share a power of two: ``codes`` float8_e4m3fn ``[..., K]`` (8 bits) or
  uint8 ``[..., K / 2]`` (4 bits e2m1, two a byte, the first in the low half), ``scales`` ``[..., K / 32]``
  float8_e8m0fnu, or uint8 of the same bytes (exponent + 127; 255 is NaN)."""
  codes: torch.Tensor
  scales: torch.Tensor

  @property
  def format(self) -> str:
    return "mxfp8" if self.codes.dtype is _FP8 else "mxfp4"

  @property
  def shape(self) -> torch.Size:
    s = self.codes.shape
    return s if self.codes.dtype is _FP8 else torch.Size((*s[:-1], 2 * s[-1]))


def _microscaled(x, name: str, what: str):
  """Checks codes and scales and returns them as rows: format, rows, K, codes, their stride, scales, their stride."""
  codes, scales = x
  dtype = codes.dtype
  eight = dtype is _FP8
  if not (eight or dtype is torch.uint8) or (scales.dtype is not _E8M0 and scales.dtype is not torch.uint8):
    raise ValueError(f"{what}: {name} must have float8_e4m3fn or packed uint8 codes and float8_e8m0fnu or uint8 scales, got "
                     f"{dtype} and {scales.dtype}")
  cs, ss = codes.shape, scales.shape
  K = (cs[-1] if eight else 2 * cs[-1]) if cs else 0
  if K < 32 or K % 32 != 0 or not ss or ss[:-1] != cs[:-1] or ss[-1] * 32 != K:
    raise ValueError(f"{what}: {name} needs a scale for each block of 32, got codes {tuple(cs)} and scales {tuple(ss)}")
  format = _lib.FORMAT_MXFP8 if eight else _lib.FORMAT_MXFP4
  if codes.is_contiguous() and scales.is_contiguous() and codes.data_ptr() % 16 == 0:
    return format, scales.numel() // ss[-1], K, codes, cs[-1], scales, ss[-1]
  c2, s2 = codes.reshape(-1, cs[-1]), scales.reshape(-1, ss[-1])
  if c2.stride(1) != 1 or c2.data_ptr() % 16 or (c2.shape[0] > 1 and (c2.stride(0) % 16 or not cs[-1] <= c2.stride(0) < 1 << 23)):
    c2 = torch.empty(c2.shape, dtype=dtype, device=c2.device).copy_(c2)
  if (ss[-1] > 1 and s2.stride(1) != 1) or (s2.shape[0] > 1 and not ss[-1] <= s2.stride(0) < 1 << 23):
    s2 = torch.empty(s2.shape, dtype=scales.dtype, device=s2.device).copy_(s2)
  R = c2.shape[0]
  return format, R, K, c2, (c2.stride(0) if R > 1 else cs[-1]), s2, (s2.stride(0) if R > 1 else ss[-1])


def _resolved(t: torch.Tensor | None) -> torch.Tensor | None:
  """t as its memory holds it: a view that is negated when read (the imaginary part of a lazily conjugated tensor) is copied."""
  return t if t is None or not t.is_neg() else t.resolve_neg()


def _empty_rows(lead, n: int, dtype: torch.dtype, dev) -> torch.Tensor:
  """``torch.empty((*lead, n))``, for a matrix in 3/5 of its host time."""
  if len(lead) == 1:
    return torch.empty_strided((lead[0], n), (n, 1), dtype=dtype, device=dev)
  return torch.empty((*lead, n), dtype=dtype, device=dev)


def _empty_microscaled(lead, K: int, format: str, dev) -> Microscaled:
  codes = _empty_rows(lead, K, _FP8, dev) if format == "mxfp8" else _empty_rows(lead, K // 2, torch.uint8, dev)
  return Microscaled(codes, _empty_rows(lead, K // 32, _E8M0, dev))


def _rows2(t: torch.Tensor, aligned: bool):
  """``[R, C]`` rows of ``[..., C]`` with a unit last stride (copied where there is none, or where 16-byte rows are asked for),
  and their stride."""
  Cn = t.shape[-1]
  if t.ndim == 2 and t.is_contiguous() and not (aligned and t.data_ptr() % 16):
    return t, Cn
  t2 = t if t.ndim == 2 else t.reshape(-1, Cn)
  if (Cn > 1 and t2.stride(1) != 1) or (aligned and (t2.data_ptr() % 16 or (t2.shape[0] > 1 and t2.stride(0) * t2.element_size() % 16))):
    t2 = torch.empty(t2.shape, dtype=t2.dtype, device=t2.device).copy_(t2)
  return t2, (t2.stride(0) if t2.shape[0] > 1 else Cn)


def mx_quantize(x: torch.Tensor, format: str = "mxfp4") -> Microscaled:
  """Microscaled numbers of ``x`` ``[..., K]``, bf16, fp16 or float32, K a multiple of 32: ``format`` ``"mxfp8"`` (e4m3) or
  ``"mxfp4"`` (e2m1).  A block's scale is ``2 ** (floor(log2(max |x|)) - 8)``, or ``- 2`` of 4 bits, from ``2 ** -127`` on;
  what it leaves is rounded to the nearest code, ties to the even one, at most 448 or 6.  A block with a NaN or an infinity is
  NaN as a whole."""
  if _front:
    result = _front.mx_quantize(x, format)
    if result is not None:
      return result
  what = "mx_quantize"
  _no_grad(what, x)
  dev = _require_cuda(x)
  if format not in _FORMATS:
    raise ValueError(f"{what}: format {format!r} is not 'mxfp8' or 'mxfp4'")
  if x.dtype not in _ELEMENT_TYPES:
    raise ValueError(f"{what}: x must be bfloat16, float16 or float32, got {x.dtype}")
  if x.ndim < 1 or not 32 <= x.shape[-1] < 1 << 31 or x.shape[-1] % 32 != 0:
    raise ValueError(f"{what}: the last dim must be a multiple of 32 below 2^31, got {tuple(x.shape)}")
  x, K = _resolved(x), x.shape[-1]
  result = _empty_microscaled(x.shape[:-1], K, format, dev)
  if x.numel() == 0:
    return result
  x2, rs = _rows2(x, True)
  a = _lib.mx_convert_args(x2.shape[0], K, _ELEMENT_TYPES[x.dtype], _FORMATS[format], x2.data_ptr(), rs, result.codes.data_ptr(),
                           result.codes.shape[-1], result.scales.data_ptr(), K // 32)
  _launch(_library().sf_hip_mx_encode_fwd, x2, "sf_hip_mx_encode_fwd", C.byref(a))
  return result


def mx_dequantize(x: Microscaled, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
  """The numbers ``[..., K]`` that codes and scales stand for, rounded once to ``dtype`` (bf16, fp16 or float32)."""
  if _front:
    result = _front.mx_dequantize(*x, dtype)
    if result is not None:
      return result
  what = "mx_dequantize"
  _no_grad(what, *x)
  _require_cuda(*x)
  if dtype not in _ELEMENT_TYPES:
    raise ValueError(f"{what}: dtype must be bfloat16, float16 or float32, got {dtype}")
  format, R, K, codes, c_rs, scales, s_rs = _microscaled(x, "x", what)
  if K >= 1 << 31:
    raise ValueError(f"{what}: rows of {K}, not below 2^31")
  out = _empty_rows(x.codes.shape[:-1], K, dtype, codes.device)
  if R == 0:
    return out
  a = _lib.mx_convert_args(R, K, _ELEMENT_TYPES[dtype], format, out.data_ptr(), K, codes.data_ptr(), c_rs, scales.data_ptr(), s_rs)
  _launch(_library().sf_hip_mx_decode_fwd, codes, "sf_hip_mx_decode_fwd", C.byref(a))
  return out


def mx_linear(x: Microscaled, w: Microscaled, bias: torch.Tensor | None = None, *, dtype: torch.dtype = torch.bfloat16,
              out: torch.Tensor | None = None) -> torch.Tensor:
  """``x @ w.T + bias`` of microscaled ``x`` ``[..., K]`` and ``w`` ``[N, K]``: ``[..., N]`` in ``dtype`` (bf16 or fp16; that of
  ``out`` where given).  8-bit x with 8- or 4-bit w, or 4-bit both.  ``bias`` ``[N]`` float32 (others are cast at every call).
  ``out`` ``[..., N]`` with a unit last stride overlaps no input.  Sums are fp32; of 8-bit codes the matrix unit adds 8
  products (8 consecutive k) at a time and cuts off what lies below 2^-13 of the largest of them."""
  if _front and out is None:
    result = _front.mx_linear(*x, *w, bias, dtype)
    if result is not None:
      return result
  what = "mx_linear"
  _no_grad(what, *x, *w, bias, out)
  dev = _require_cuda(*x, *w, bias, out)
  if w.codes.ndim != 2:
    raise ValueError(f"{what}: w must be [features, K], got codes {tuple(w.codes.shape)}")
  xf, M, K, xc, x_rs, xs, xs_rs = _microscaled(x, "x", what)
  wf, N, Kw, wc, w_rs, ws, ws_rs = _microscaled(w, "w", what)
  if Kw != K or N < 1 or N > 1 << 24 or K > 1 << 22 or M >= 1 << 31:
    raise ValueError(f"{what}: x [{M}, {K}] (up to 2^22) against w [{N}, {Kw}] (up to 2^24 rows)")
  if xf == _lib.FORMAT_MXFP4 and wf == _lib.FORMAT_MXFP8:
    raise ValueError(f"{what}: 4-bit x takes 4-bit w")
  if bias is not None:
    if bias.shape != (N,):
      raise ValueError(f"{what}: bias must be [{N}], got {tuple(bias.shape)}")
    bias = _resolved(bias)
    if bias.dtype is not torch.float32 or not bias.is_contiguous():
      bias = _f32(bias)
  shape = (*x.codes.shape[:-1], N)
  if out is None:
    if dtype not in (torch.bfloat16, torch.float16):
      raise ValueError(f"{what}: dtype must be bfloat16 or float16, got {dtype}")
    y = result = _empty_rows(shape[:-1], N, dtype, dev)
    y_rs = N
  else:
    dtype = out.dtype
    if out.is_neg():
      raise ValueError(f"{what}: out is a view that is negated when read")
    if out.shape != shape or dtype not in (torch.bfloat16, torch.float16) or (N > 1 and out.stride(-1) != 1):
      raise ValueError(f"{what}: out must be bfloat16 or float16 {shape} with a unit last stride, got {dtype} {tuple(out.shape)}")
    result = out
    try:
      y = out if out.ndim == 2 else out.view(-1, N)
    except RuntimeError:
      raise ValueError(f"{what}: the leading dims of out must be one stride apart") from None
    y_rs = y.stride(0) if M > 1 else N
    if y_rs < N:
      raise ValueError(f"{what}: out must hold every element once")
    y0 = y.data_ptr()
    y1 = y0 + (2 * ((M - 1) * y_rs + N) if M > 0 else 0)
    for t in (xc, xs, wc, ws, bias):
      if t is not None:
        t0, t1 = _span(t)
        if t0 < y1 and y0 < t1:
          raise ValueError(f"{what}: out overlaps an input")
  if M == 0:
    return result
  a = _lib.mx_linear_args(M, N, K, xf, wf, _ELEMENT_TYPES[dtype], xc.data_ptr(), x_rs, xs.data_ptr(), xs_rs, wc.data_ptr(), w_rs,
                          ws.data_ptr(), ws_rs, _vp(bias) or 0, y.data_ptr(), y_rs)
  lib = _library()
  ref = C.byref(a)
  need = lib.sf_hip_mx_linear_workspace_bytes(ref)
  work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
  _launch(lib.sf_hip_mx_linear_fwd, xc, "sf_hip_mx_linear_fwd", ref, _vp(work), need)
  _written(out)
  return result


def _norm_outputs(what, shape, dtype, R, inputs, weight, aligned, outs):
  """Checks given outputs of the norm (None: not given) against the inputs' rows, (pointer, row stride); returns the pointer and
  row stride of each."""
  Cn = shape[-1]
  size = 4 if dtype is torch.float32 else 2
  width, rows = Cn * size, []

  def apart(p, sp, q, sq):
    """Whether rows lie apart: separate ranges, or separate columns of rows of one width."""
    sp, sq = sp * size, sq * size
    if p + (R - 1) * sp + width <= q or q + (R - 1) * sq + width <= p:
      return True
    return sp == sq and width <= sp and width <= (p - q) % sp <= sp - width

  for o, name in zip(outs, ("out", "out_sum")):
    if o is None:
      continue
    if o.is_neg():
      raise ValueError(f"{what}: {name} is a view that is negated when read")
    if o.shape != shape or o.dtype is not dtype or (Cn > 1 and o.stride(-1) != 1):
      raise ValueError(f"{what}: {name} must be {dtype} {tuple(shape)} with a unit last stride")
    try:
      o2 = o if o.ndim == 2 else o.view(-1, Cn)
    except RuntimeError:
      raise ValueError(f"{what}: the leading dims of {name} must be one stride apart") from None
    p, st = o2.data_ptr(), o2.stride(0) if R > 1 else Cn
    if st < Cn:
      raise ValueError(f"{what}: {name} must hold every element once")
    if aligned and (p % 16 or st * size % 16):
      raise ValueError(f"{what}: {name} must lie in 16-byte aligned rows with a microscaled output")
    if R > 0:
      if not all((p == q and (st == sq or R == 1)) or apart(p, st, q, sq) for q, sq in inputs):
        raise ValueError(f"{what}: outputs may be x or residual itself, and overlap nothing else")
      if weight is not None and not (p + (R - 1) * st * size + width <= weight.data_ptr() or weight.data_ptr() + 4 * Cn <= p):
        raise ValueError(f"{what}: an output overlaps the weight")
    rows.append((p, st))
  if R > 0 and len(rows) == 2 and not apart(*rows[0], *rows[1]):
    raise ValueError(f"{what}: out and out_sum overlap")
  return rows


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, *, eps: float = 1e-6,
                 output: str | None = None, out: torch.Tensor | None = None,
                 out_sum: torch.Tensor | None = None) -> tuple[torch.Tensor | Microscaled, torch.Tensor | None]:
  """``h = x + residual`` and its root-mean-square norm ``h rsqrt(mean h^2 + eps) weight`` over the last dim; returns the
  norm and h (None without a residual: h is x).

  ``x`` and ``residual`` ``[..., C]``, bf16, fp16 or float32 (one type), any C and strides; h is rounded to the type, the norm is of
  the rounded h, formed in 64 bits and rounded once.  ``weight`` ``[C]`` float32 (others are cast at every call; None: 1).
  ``output`` ``"mxfp8"`` or ``"mxfp4"``: the norm microscaled, as ``mx_quantize`` of the unrounded norm, for ``mx_linear``; C a multiple
  of 32 then.

  ``out`` (without ``output``) and ``out_sum`` like x with a unit last stride; each may be ``x`` or ``residual`` itself, and
  overlaps nothing else."""
  if _front and out is None and out_sum is None:
    result = _front.add_rms_norm(x, residual, weight, eps, output)
    if result is not None:
      return result
  what = "add_rms_norm"
  _no_grad(what, x, residual, weight, out, out_sum)
  dev = _require_cuda(x, residual, weight, out, out_sum)
  dtype, shape = x.dtype, x.shape
  if dtype not in _ELEMENT_TYPES or (residual is not None and (residual.dtype is not dtype or residual.shape != shape)):
    raise ValueError(f"{what}: x and residual must be bfloat16, float16 or float32 of one type and shape, got {dtype} {tuple(shape)}"
                     f"{'' if residual is None else f' and {residual.dtype} {tuple(residual.shape)}'}")
  if len(shape) < 1 or not 0 < shape[-1] < 1 << 30:
    raise ValueError(f"{what}: x must be [..., C], got {tuple(shape)}")
  Cn = shape[-1]
  if output is not None and (output not in _FORMATS or Cn % 32 != 0):
    raise ValueError(f"{what}: output {output!r} is not None, 'mxfp8' or 'mxfp4', or {Cn} no multiple of 32")
  if (output is not None and out is not None) or (residual is None and out_sum is not None):
    raise ValueError(f"{what}: out goes without output, out_sum with a residual")
  if not 0.0 <= eps <= 1e30:
    raise ValueError(f"{what}: eps {eps} is not finite and >= 0, or above 1e30")
  if weight is not None:
    if weight.shape != (Cn,):
      raise ValueError(f"{what}: weight must be [{Cn}], got {tuple(weight.shape)}")
    weight = _resolved(weight)
    if weight.dtype is not torch.float32 or not weight.is_contiguous():
      weight = _f32(weight)
  x, residual, aligned = _resolved(x), _resolved(residual), output is not None
  x2, x_rs = _rows2(x, aligned)
  R, x_p = x2.shape[0], x2.data_ptr()
  r2, r_p, r_rs = None, 0, 0
  if residual is not None:
    r2, r_rs = _rows2(residual, aligned)
    r_p = r2.data_ptr()
  y_p, y_rs, h_p, h_rs, total, codes = 0, 0, 0, 0, out_sum, None
  if out is not None or out_sum is not None:
    rows = _norm_outputs(what, shape, dtype, R, ((x_p, x_rs),) if r2 is None else ((x_p, x_rs), (r_p, r_rs)), weight, aligned, (out, out_sum))
    if out is not None:
      y_p, y_rs = rows[0]
    if out_sum is not None:
      h_p, h_rs = rows[-1]
  if output is not None:
    result = codes = _empty_microscaled(shape[:-1], Cn, output, dev)
  elif out is None:
    result = _fresh(x)
    y_p, y_rs = result.data_ptr(), Cn
  else:
    result = out
  if residual is not None and out_sum is None:
    total = _fresh(x)
    h_p, h_rs = total.data_ptr(), Cn
  if R == 0:
    return result, total
  a = _lib.add_rms_norm_args(R, Cn, _ELEMENT_TYPES[dtype], 0 if output is None else _FORMATS[output], eps, x_p, x_rs, r_p, r_rs,
                             _vp(weight) or 0, h_p, h_rs, y_p, y_rs,
                             *((0, 0, 0, 0) if codes is None else
                               (codes.codes.data_ptr(), codes.codes.shape[-1], codes.scales.data_ptr(), Cn // 32)))
  _launch(_library().sf_hip_add_rms_norm_fwd, x2, "sf_hip_add_rms_norm_fwd", C.byref(a))
  _written(out, out_sum)
  return result, total
