"""Cases that time the operators of a serving step: the residual's addition with the root-mean-square
norm, microscaled numbers (blocks of 32 elements of 8 or 4 bits with a power of two each: quantisation
and the product), and a paged cache of keys and values (writing new tokens, attention of new tokens
over it).

``own`` chooses the side: False computes an operator in its plain form, elementary torch operations
in 32 bits (the norm that is rounded to 8 or 4 bits in 64: its values lie next to borders), True makes
the framework's calls.  Lengths of a case are texts of numbers, one per sequence.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
BLOCK = 32
# largest magnitude and exponent of the largest power of two of an element
_ELEMENT = {"mxfp8": (448.0, 8), "mxfp4": (6.0, 2)}
_BITS = {"mxfp8": 8, "mxfp4": 4}


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------

def _named(name, case):
  return {"name": name, **case} if name else case


def _norm(name, rows, dim, dtype, residual, output):
  """``output``: the input's type, or microscaled for a product."""
  return _named(name, {"op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "output": output})


def _quantize(name, rows, dim, dtype, format):
  """8 bits: codes and scales.  4 bits: the values that they stand for, so there and back."""
  return _named(name, {"op": "quantize", "rows": rows, "dim": dim, "dtype": dtype, "format": format})


def _linear(name, rows, dim, features, x_format, w_format, bias, dtype):
  return _named(name, {"op": "linear", "rows": rows, "dim": dim, "features": features, "x_format": x_format,
                       "w_format": w_format, "bias": bias, "dtype": dtype})


def _paged(name, op, lens_q, lens_k, heads, kv_heads, dim, page, dtype):
  """``lens_k`` count the new tokens of ``lens_q`` too."""
  case = {"op": op, "lens_q": " ".join(map(str, lens_q)), "lens_k": " ".join(map(str, lens_k)), "kv_heads": kv_heads,
          "dim": dim, "page": page, "dtype": dtype}
  if op == "attention":
    case["heads"] = heads
  return _named(name, case)


def listed():
  depths = [8192, 37, 2500, 1024, 3333, 1, 4000, 700, 5120, 16, 33, 7001, 129, 2048, 6000, 450,
            4096, 999, 64, 300, 1777, 2900, 8191, 511, 1200, 15, 3600, 800, 5555, 256, 100, 1500]
  pieces, before = [2048, 1, 517, 1300, 33, 1024, 259, 1777], [2048, 4000, 0, 1, 900, 1024, 31, 515]
  return [
      # the norm between two layers: one token of each of 8 sequences, and a long prompt whose next product takes 8 bits
      _norm("norm_tokens_8", 8, 4096, "bf16", True, "same"),
      _norm("norm_prompt_16384_mxfp8", 16384, 4096, "bf16", True, "mxfp8"),
      # activations of a few tokens to 8 bits, and a layer's weights to 4 bits and what became of them
      _quantize("quantize_rows_37_mxfp8", 37, 768, "bf16", "mxfp8"),
      _quantize("quantize_weights_mxfp4", 16384, 4096, "bf16", "mxfp4"),
      # products: a token of each of 8 sequences, a ragged batch of prompts, the largest
      _linear("linear_tokens_8", 8, 4096, 12288, "mxfp8", "mxfp4", False, "bf16"),
      _linear("linear_ragged_777", 777, 4096, 4096, "mxfp8", "mxfp8", True, "fp16"),
      _linear("linear_8192", 8192, 8192, 8192, "mxfp4", "mxfp4", False, "bf16"),
      # new keys and values into their pages: one token of each of 64 sequences, pieces of prompts
      _paged("write_tokens_64", "write", [1] * 64, [1 + 61 * i for i in range(64)], 0, 8, 128, 16, "bf16"),
      _paged("write_pieces_ragged", "write", pieces, [a + b for a, b in zip(pieces, before)], 0, 8, 128, 64, "fp16"),
      # one token of each of 32 sequences over caches of very different lengths
      _paged("attention_tokens_32", "attention", [1] * 32, depths, 32, 8, 128, 16, "bf16"),
      # a step that takes a piece of one prompt along with the tokens of others
      _paged("attention_piece_and_tokens", "attention", [512] + [1] * 12, [6000] + depths[2:14], 16, 2, 64, 32, "fp16"),
      # a long piece of a prompt whose beginning is in the cache
      _paged("attention_piece_4096_of_16384", "attention", [4096], [16384], 32, 8, 128, 64, "bf16"),
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["norm", "quantize", "linear", "linear", "write", "attention", "attention", "attention"])
  if op in ("norm", "quantize"):
    dtype, dim = rng.choice(["bf16", "bf16", "fp16", "fp32"]), BLOCK * _log_int(rng, 3, 256)
    rows = _log_int(rng, 1, (1 << 25) // dim)
    if op == "quantize":
      return _quantize(None, rows, dim, dtype, rng.choice(["mxfp8", "mxfp4"]))
    output = rng.choice(["same", "same", "mxfp8", "mxfp4"])
    return _norm(None, rows, dim - (rng.randrange(8) if output == "same" else 0), dtype, rng.random() < 0.75, output)
  if op == "linear":
    x, w = rng.choice([("mxfp8", "mxfp4"), ("mxfp8", "mxfp8"), ("mxfp4", "mxfp4")])
    dim, features = BLOCK * _log_int(rng, 4, 256), _log_int(rng, 64, 8192)
    return _linear(None, _log_int(rng, 1, 8192), dim, features - features % rng.choice([1, 8, 64]), x, w, rng.random() < 0.4,
                   rng.choice(["bf16", "bf16", "fp16"]))
  kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 8])
  dim, page, dtype = rng.choice([32, 64, 64, 80, 96, 128, 128]), rng.choice([16, 16, 32, 64, 64, 128, 48]), rng.choice(["bf16", "fp16"])
  if op == "write":
    count, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 512)
    lens_q = [_log_int(rng, 1, longest) for _ in range(count)]
    return _paged(None, op, lens_q, [n + _log_int(rng, 1, 2048) - 1 for n in lens_q], 0, kv_heads, dim, page, dtype)
  kind = rng.choice(["tokens", "piece", "mixed"])
  count = 1 if kind == "piece" else _log_int(rng, 1, 32)
  # (padded to the longest sequence, the plain form stays within some GB)
  longest = _log_int(rng, 16, min(16384, (1 << 27) // (count * kv_heads * dim)))
  lens_k = [_log_int(rng, 1, longest) for _ in range(count)]
  lens_q = [1] * count
  if kind != "tokens":
    most = max(2, min(2048, (1 << 28) // (count * kv_heads * group * longest)))
    lens_q[0] = _log_int(rng, 2, most)
    lens_k[0] = max(lens_k[0], lens_q[0])
  return _paged(None, op, lens_q, lens_k, kv_heads * group, kv_heads, dim, page, dtype)


def _lens(text):
  return [int(x) for x in text.split()]


# ---------------------------------------------------------------------------------------
# Microscaled numbers in their plain form.  A block of 32 elements x has the scale 2^e,
# e = max(floor(log2 max |x|) - E, -127) with E the exponent of the element type's largest power of two, and
# the codes of x 2^-e, rounded to the nearest (ties to the even code), at most the type's largest.
# 8 bits: 4 of exponent, 3 of mantissa; 4 bits: 2 and 1, two codes a byte, the first in the low half.
# Scales are bytes, e + 127.
# ---------------------------------------------------------------------------------------

def _plain_quantize(x, format):
  """Codes as float8, or as the values of 4 bits; scales as bytes; both of blocks [..., K / 32, 32]."""
  largest, power = _ELEMENT[format]
  x = x.unflatten(-1, (-1, BLOCK))
  top = x.abs().amax(-1, keepdim=True)
  byte = torch.where(top == 0, 0, (torch.frexp(top).exponent - 1 - power + 127).clamp(0, 254))
  y = (x * _powers(x.device, 127)[(254 - byte).long()].to(x.dtype)).clamp(-largest, largest)
  if format == "mxfp8":
    # (one rounding: from 64 bits by way of 32 with the last bit set where something was cut off)
    y = _cut(y).to(torch.float8_e4m3fn)
  else:
    step = torch.where(y.abs() >= 4, 2.0, torch.where(y.abs() >= 2, 1.0, 0.5)).to(y.dtype)
    y = (y / step).round() * step
  return y, byte.to(torch.uint8)


def _cut(y):
  if y.dtype == torch.float32:
    return y
  z = y.float()
  z = torch.where(z.double().abs() > y.abs(), torch.nextafter(z, torch.zeros_like(z)), z)
  return torch.where(z.double() != y, (z.view(torch.int32) | 1).view(torch.float32), z)


def _powers(device, bias):
  """2^(byte - bias) of each byte, 64 bits."""
  return torch.tensor([2.0 ** (i - bias) for i in range(255)] + [math.nan], dtype=torch.float64, device=device)


def _plain_values(codes, scales, dtype):
  """What codes and scales stand for: [..., K]."""
  if codes.dtype == torch.uint8:
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=dtype, device=codes.device)
    table = torch.cat((table, -table))
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    values = table[both.int()]
  else:
    values = codes.to(dtype)
  return (values.unflatten(-1, (-1, BLOCK)) * _powers(codes.device, 127).to(dtype)[scales.int()].unsqueeze(-1)).flatten(-2)


def _packed(values):
  """The bytes of values that 4 bits hold."""
  m = values.abs()
  code = torch.where(m <= 2, 2 * m, torch.where(m <= 4, m + 2, m / 2 + 4)).to(torch.uint8) | (torch.signbit(values).to(torch.uint8) << 3)
  pairs = code.unflatten(-1, (-1, 2))
  return pairs[..., 0] | (pairs[..., 1] << 4)


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _offsets(lens):
  return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
  gen = torch.Generator(device="cuda").manual_seed(seed)

  def normal(*shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

  def channels(rows, dim):
    """Activations: some channels are much larger than the others."""
    return normal(rows, dim) * (0.5 * normal(dim)).exp_()

  def microscaled(x, format):
    values, scales = _plain_quantize(x, format)
    codes = values.flatten(-2) if format == "mxfp8" else _packed(values.flatten(-2))
    return codes, scales.squeeze(-1)

  state = {"case": case}
  dtype = _TYPES[case["dtype"]]
  if case["op"] == "norm":
    state.update(x=channels(case["rows"], case["dim"]).to(dtype), weight=1.0 + 0.2 * normal(case["dim"]),
                 residual=(4.0 * normal(case["rows"], case["dim"])).to(dtype) if case["residual"] else None)
  elif case["op"] == "quantize":
    state.update(x=(0.02 * channels(case["rows"], case["dim"])).to(dtype))
  elif case["op"] == "linear":
    x_codes, x_scales = microscaled(channels(case["rows"], case["dim"]), case["x_format"])
    w_codes, w_scales = microscaled(normal(case["features"], case["dim"]) * case["dim"] ** -0.5, case["w_format"])
    state.update(x_codes=x_codes, x_scales=x_scales, w_codes=w_codes, w_scales=w_scales,
                 bias=normal(case["features"]) if case["bias"] else None)
  else:
    lens_q, lens_k, page, hk, d = _lens(case["lens_q"]), _lens(case["lens_k"]), case["page"], case["kv_heads"], case["dim"]
    needed = [-(-n // page) for n in lens_k]
    total = sum(needed)
    # pages of all sequences in the order in which they were handed out, some of the cache free
    free = torch.randperm(total + total // 8 + 1, generator=gen, device="cuda").to(torch.int32)
    owner = torch.cat([torch.full((n,), b) for b, n in enumerate(needed)])
    slot = torch.cat([torch.arange(n) for n in needed])
    table = torch.zeros(len(lens_k), max(needed), dtype=torch.int32, device="cuda")
    table[owner.cuda(), slot.cuda()] = free[:total]
    pages = (free.numel(), page, hk, d)
    state.update(k_pages=normal(*pages).to(dtype), v_pages=normal(*pages).to(dtype), table=table, cu=_offsets(lens_q),
                 len_k=torch.tensor(lens_k, dtype=torch.int32).cuda(), longest=max(lens_k))
    tokens = sum(lens_q)
    if case["op"] == "write":
      # as the projection left them: columns of one buffer
      fused = normal(tokens, 2 * hk, d).to(dtype)
      state.update(k=fused[:, :hk], v=fused[:, hk:])
    else:
      state.update(q=normal(tokens, case["heads"], d).to(dtype), most=max(lens_q))
  return state


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------

def _plain_norm(state):
  case, x = state["case"], state["x"]
  total = None
  if state["residual"] is not None:
    total = x = (x.float() + state["residual"].float()).to(x.dtype)
  wide = x.float() if case["output"] == "same" else x.double()
  y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + EPS) * state["weight"].to(wide.dtype)
  if case["output"] == "same":
    return {"y": y.to(x.dtype), "sum": total}
  return {**_plain_coded(y, case["output"]), "sum": total}


def _plain_coded(x, format):
  codes, scales = _plain_quantize(x, format)
  if format == "mxfp8":
    return {"codes": codes.flatten(-2), "scales": scales.squeeze(-1).view(torch.float8_e8m0fnu)}
  return {"values": (codes * _powers(x.device, 127)[scales.long()].to(codes.dtype)).flatten(-2).to(torch.bfloat16)}


def _plain_linear(state):
  x, w = (_plain_values(state[n + "_codes"], state[n + "_scales"], torch.float32) for n in ("x", "w"))
  y = torch.matmul(x, w.t())
  if state["bias"] is not None:
    y = y + state["bias"]
  return y.to(_TYPES[state["case"]["dtype"]])


def _plain_write(state):
  case, cu, table = state["case"], state["cu"].long(), state["table"].long()
  token = torch.arange(state["k"].shape[0], device=cu.device)
  b = torch.searchsorted(cu, token, right=True) - 1
  at = state["len_k"].long()[b] - (cu[b + 1] - token)
  page, row = table[b, at // case["page"]], at % case["page"]
  state["k_pages"][page, row] = state["k"]
  state["v_pages"][page, row] = state["v"]
  return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _plain_attention(state):
  """All sequences at once, padded to the longest."""
  case, q, cu = state["case"], state["q"], state["cu"].long()
  h, hk, d = case["heads"], case["kv_heads"], case["dim"]
  n, m, most, longest = cu[1:] - cu[:-1], state["len_k"].long(), state["most"], state["longest"]
  k, v = (state[name][state["table"].long()].flatten(1, 2)[:, :longest].float().transpose(1, 2) for name in ("k_pages", "v_pages"))
  i, j = torch.arange(most, device=q.device), torch.arange(longest, device=q.device)
  rows = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
  qs = q[rows].float().unflatten(2, (hk, h // hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)                  # [B, hk, g n, d]
  s = torch.matmul(qs, k.transpose(2, 3)).unflatten(2, (h // hk, most)) * (1.0 / math.sqrt(d))
  s.masked_fill_((j > i[:, None] + (m - n)[:, None, None])[:, None, None], -math.inf)
  s -= s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
  p = s.exp_()
  total = p.sum(-1, keepdim=True)
  p /= torch.where(total == 0, torch.ones_like(total), total)
  o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (h // hk, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, n, h, d]
  return o[i < n[:, None]].to(q.dtype)


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------

def run(state):
  case = state["case"]
  op = case["op"]
  if not own:
    if op == "norm":
      return _plain_norm(state)
    if op == "quantize":
      return _plain_coded(state["x"].float(), case["format"])
    return {"linear": _plain_linear, "write": _plain_write, "attention": _plain_attention}[op](state)
  from sparsefold_amd.backends.hip import ops
  if op in ("norm", "quantize"):
    if op == "norm":
      output = None if case["output"] == "same" else case["output"]
      y, total = ops.add_rms_norm(state["x"], state["residual"], state["weight"], eps=EPS, output=output)
      result = {"sum": total}
      if output is None:
        return {"y": y, **result}
    else:
      output, result = case["format"], {}
      y = ops.mx_quantize(state["x"], output)
    if output == "mxfp8":
      return {"codes": y.codes, "scales": y.scales, **result}
    return {"values": ops.mx_dequantize(y, torch.bfloat16), **result}
  if op == "linear":
    return ops.mx_linear(ops.Microscaled(state["x_codes"], state["x_scales"]), ops.Microscaled(state["w_codes"], state["w_scales"]),
                         state["bias"], dtype=_TYPES[case["dtype"]])
  pages = (state["k_pages"], state["v_pages"], state["table"])
  if op == "write":
    ops.paged_cache_write(state["k"], state["v"], *pages, state["cu"], state["len_k"])
    return {"k_pages": pages[0], "v_pages": pages[1]}
  return ops.paged_attention(state["q"], *pages, state["cu"], state["len_k"], causal=True, max_len=state["longest"])


# ---------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------

def work(case):
  op, size = case["op"], _SIZES[case["dtype"]]
  if op in ("norm", "quantize"):
    n, output = case["rows"] * case["dim"], case.get("output") or case["format"]
    coded = 0 if output == "same" else n * _BITS[output] // 8 + n // BLOCK
    if op == "quantize":
      # 4 bits come back as 16: the codes are written and read again
      return {"bytes": n * size + coded + (n * 2 + coded if output == "mxfp4" else 0), "flops": 3 * n}
    values = n * size if output == "same" else coded + (n * 2 + coded if output == "mxfp4" else 0)
    return {"bytes": n * size * (3 if case["residual"] else 1) + values + 4 * case["dim"],
            "flops": n * (5 if case["residual"] else 4) + (0 if output == "same" else 3 * n)}
  if op == "linear":
    m, k, n = case["rows"], case["dim"], case["features"]
    codes = (m * _BITS[case["x_format"]] + n * _BITS[case["w_format"]]) * k // 8 + (m + n) * (k // BLOCK)
    return {"bytes": codes + m * n * size + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
  lens_q, lens_k, hk, d = _lens(case["lens_q"]), _lens(case["lens_k"]), case["kv_heads"], case["dim"]
  if op == "write":
    return {"bytes": 4 * size * sum(lens_q) * hk * d, "flops": 0}
  h = case["heads"]
  pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(lens_q, lens_k))
  return {"bytes": size * d * (2 * sum(lens_q) * h + 2 * sum(lens_k) * hk), "flops": 4 * d * h * pairs}


# ---------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------

def _grid(format):
  """Every non-negative value of an element, in the order of the codes."""
  bits, bias = (3, 7) if format == "mxfp8" else (1, 1)
  found = []
  for code in range(127 if format == "mxfp8" else 8):
    e, f = code >> bits, code & ((1 << bits) - 1)
    found.append(math.ldexp(f, 1 - bias - bits) if e == 0 else math.ldexp((1 << bits) + f, e - bias - bits))
  return found


def _exact_codes(x, format):
  """Elements and scales of x, both as 64-bit values."""
  grid = torch.tensor(_grid(format), dtype=torch.float64, device=x.device)
  blocks = x.to(torch.float64).reshape(*x.shape[:-1], -1, BLOCK)
  top = blocks.abs().max(dim=-1, keepdim=True).values
  mantissa, e = torch.frexp(top)                                       # top = mantissa 2^e, 1/2 <= mantissa < 1
  e = torch.where(top > 0, e - 1 - int(math.log2(grid[-1].item())), -127).clamp(min=-127)
  scale = torch.tensor([math.ldexp(1.0, i) for i in range(-127, 128)], dtype=torch.float64, device=x.device)[(e + 127).long()]
  size = blocks.abs() / scale
  middle = (grid[1:] + grid[:-1]) / 2
  below, through = torch.searchsorted(middle, size), torch.searchsorted(middle, size, right=True)
  code = torch.where(below == through, below, below + (below & 1))      # on a border: the even code
  return torch.copysign(grid[code], blocks).flatten(-2), scale.squeeze(-1)


def _exact_rows(state):
  case, x, result = state["case"], state["x"].to(torch.float64), {}
  if case["op"] == "norm":
    if state["residual"] is not None:
      result["sum"] = x + state["residual"].to(torch.float64)
      x = result["sum"].to(_TYPES[case["dtype"]]).to(torch.float64)
    else:
      result["sum"] = None
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * state["weight"].to(torch.float64)
    if case["output"] == "same":
      return {"y": x, **result}
  format = case.get("output") or case["format"]
  element, scale = _exact_codes(x, format)
  if format == "mxfp8":
    return {"codes": element, "scales": scale, **result}
  return {"values": element * scale.repeat_interleave(BLOCK, dim=-1), **result}


def _exact_linear(state):
  def decode(codes, scales, format):
    grid = _grid(format)
    table = torch.tensor(grid + ([math.nan] if format == "mxfp8" else []), dtype=torch.float64, device="cuda")
    table = torch.cat((table, -table))
    byte = codes.view(torch.uint8).to(torch.int64)
    if format == "mxfp4":
      byte = torch.stack((byte % 16, byte // 16), dim=-1).reshape(byte.shape[0], -1)
    powers = torch.tensor([math.ldexp(1.0, i - 127) for i in range(256)], dtype=torch.float64, device="cuda")
    return table[byte] * powers[scales.to(torch.int64)].repeat_interleave(BLOCK, dim=1)

  case = state["case"]
  result = decode(state["x_codes"], state["x_scales"], case["x_format"]) @ decode(state["w_codes"], state["w_scales"], case["w_format"]).T
  return result if state["bias"] is None else result + state["bias"].to(torch.float64)


def _exact_paged(state):
  case, table = state["case"], state["table"].tolist()
  page, group = case["page"], case.get("heads", 0) // case["kv_heads"]
  k_pages, v_pages = state["k_pages"].to(torch.float64), state["v_pages"].to(torch.float64)
  if case["op"] == "attention":
    q = state["q"].to(torch.float64)
    result = torch.zeros_like(q)
  first = 0
  for b, (n, m) in enumerate(zip(_lens(case["lens_q"]), _lens(case["lens_k"]))):
    last = first + n
    mine = table[b][:-(-m // page)]
    if case["op"] == "write":
      at = m - n
      while at < m:                                                    # a page's part at a time
        count = min(page - at % page, m - at)
        token = last - (m - at)
        for pages, new in ((k_pages, state["k"]), (v_pages, state["v"])):
          pages[mine[at // page], at % page:at % page + count] = new[token:token + count].to(torch.float64)
        at += count
    else:
      keys, values = (torch.cat([pages[p] for p in mine])[:m] for pages in (k_pages, v_pages))
      seen = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(diagonal=m - n)
      for head in range(case["heads"]):
        logits = q[first:last, head] @ keys[:, head // group].contiguous().T * case["dim"] ** -0.5
        weights = torch.softmax(logits.masked_fill(~seen, -math.inf), dim=-1)
        result[first:last, head] = torch.nan_to_num(weights, nan=0.0) @ values[:, head // group].contiguous()
    first = last
  return {"k_pages": k_pages, "v_pages": v_pages} if case["op"] == "write" else result


def exact(case, seed):
  state = prepare(case, seed)
  if case["op"] in ("norm", "quantize"):
    return _exact_rows(state)
  return _exact_linear(state) if case["op"] == "linear" else _exact_paged(state)
