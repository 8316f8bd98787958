"""Refused arguments of the packed-sequence calls, and the set-up of rotary frequencies; nothing here
launches a kernel."""
import ctypes as C
import math

import pytest
import torch

from sparsefold_amd import _lib
from sparsefold_amd.backends.hip import ops

BF = torch.bfloat16


class _Launched(Exception):
  pass


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
  """Argument checks run on host tensors; reaching the library ends the call."""
  def refuse():
    raise _Launched
  monkeypatch.setattr(ops, "_require_cuda", lambda *t: torch.device("cpu"))
  monkeypatch.setattr(ops._lib, "load", refuse)


def attention_args(**kw):
  a = dict(q=torch.zeros(6, 4, 32, dtype=BF), k=torch.zeros(6, 2, 32, dtype=BF), v=torch.zeros(6, 2, 32, dtype=BF),
           cu_q=torch.tensor([0, 2, 6], dtype=torch.int32))
  a.update(kw)
  return a


def test_device_tensors_are_needed(monkeypatch):
  monkeypatch.undo()
  with pytest.raises(ValueError, match="device tensors"):
    ops.packed_attention(**attention_args())
  with pytest.raises(ValueError, match="device tensors"):
    ops.rotary(torch.zeros(2, 1, 8), None, torch.arange(2), ops.rotary_frequencies(8))


def test_accepted_arguments_reach_the_library():
  with pytest.raises(_Launched):
    ops.packed_attention(**attention_args())
  with pytest.raises(_Launched):
    ops.packed_attention(**attention_args(cu_k=torch.tensor([0, 0, 6], dtype=torch.int32), len_k=torch.tensor([0, 3], dtype=torch.int32)))
  with pytest.raises(_Launched):
    ops.packed_attention(**attention_args(out=torch.zeros(6, 4, 64, dtype=BF)[..., 32:]))


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(6, 128, dtype=BF)), "tokens, heads, dim"),
    (dict(k=torch.zeros(6, 2, 64, dtype=BF)), "shapes"),
    (dict(v=torch.zeros(5, 2, 32, dtype=BF)), "shapes"),
    (dict(k=torch.zeros(6, 3, 32, dtype=BF), v=torch.zeros(6, 3, 32, dtype=BF)), "evenly"),
    (dict(k=torch.zeros(6, 0, 32, dtype=BF), v=torch.zeros(6, 0, 32, dtype=BF)), "evenly"),
    (dict(q=torch.zeros(6, 4, 32)), "bfloat16 or all float16"),
    (dict(k=torch.zeros(6, 2, 32, dtype=torch.float16)), "bfloat16 or all float16"),
    (dict(cu_q=torch.tensor([0, 2, 6])), "int32"),
    (dict(cu_q=torch.tensor([0], dtype=torch.int32)), "two offsets"),
    (dict(cu_k=torch.tensor([0, 6], dtype=torch.int32)), "cu_k must be int32"),
    (dict(len_q=torch.tensor([1], dtype=torch.int32)), "len_q must be int32"),
    (dict(len_k=torch.tensor([1.0, 2.0])), "len_k must be int32"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(out=torch.zeros(6, 4, 32)), "out must be"),
    (dict(out=torch.zeros(6, 4, 33, dtype=BF)[..., 1:]), "out must be"),
])
def test_attention_refuses(kw, match):
  with pytest.raises(ValueError, match=match):
    ops.packed_attention(**attention_args(**kw))


@pytest.mark.parametrize("D", [0, 4, 20, 136, 256])
def test_attention_refuses_head_dims(D):
  t = torch.zeros(6, 2, D, dtype=BF)
  with pytest.raises(ValueError, match="multiple of 8 up to 128"):
    ops.packed_attention(t, t, t, torch.tensor([0, 6], dtype=torch.int32))


def test_attention_refuses_overlaps_and_gradients():
  x = torch.zeros(6, 6, 32, dtype=BF)
  q, k, v = x[:, :2], x[:, 2:4], x[:, 4:]
  cu = torch.tensor([0, 6], dtype=torch.int32)
  for out in (q, k, v, x[:, 1:3]):
    with pytest.raises(ValueError, match="overlaps"):
      ops.packed_attention(q, k, v, cu, out=out)
  wide = torch.zeros(6, 8, 32, dtype=BF)
  with pytest.raises(_Launched):                     # other columns of the same rows
    ops.packed_attention(wide[:, :2], wide[:, 2:4], wide[:, 4:6], cu, out=wide[:, 6:])
  leaf = torch.zeros(6, 2, 32, dtype=BF, requires_grad=True)
  with pytest.raises(ValueError, match="no backward"):
    ops.packed_attention(leaf, k, v, cu)
  with torch.no_grad(), pytest.raises(_Launched):
    ops.packed_attention(leaf, k, v, cu)


def test_outputs_that_hold_an_element_twice_are_refused():
  for out in (torch.zeros(1, 4, 32, dtype=BF).expand(6, 4, 32), torch.zeros(6, 1, 32, dtype=BF).expand(6, 4, 32),
              torch.zeros(448, dtype=BF).as_strided((6, 4, 32), (64, 32, 1))):
    with pytest.raises(ValueError, match="apart from each other"):
      ops.packed_attention(**attention_args(out=out))
    q = torch.zeros(6, 4, 32, dtype=BF)
    with pytest.raises(ValueError, match="every element once"):
      ops.rotary(q, None, torch.arange(6), ops.rotary_frequencies(32), out_q=out)
    with pytest.raises(ValueError, match="every element once"):
      ops.rotary(out, None, torch.arange(6), ops.rotary_frequencies(32), out_q=out)
  with pytest.raises(_Launched):                     # head-major
    ops.packed_attention(**attention_args(out=torch.zeros(4, 6, 32, dtype=BF).transpose(0, 1)))


def test_outputs_that_expect_a_gradient_are_refused():
  leaf = torch.zeros(6, 4, 32, dtype=BF, requires_grad=True)
  with pytest.raises(ValueError, match="no backward"):
    ops.packed_attention(**attention_args(out=leaf))
  with pytest.raises(ValueError, match="no backward"):
    ops.rotary(torch.zeros(6, 4, 32, dtype=BF), None, torch.arange(6), ops.rotary_frequencies(32), out_q=leaf)


def test_scalars_past_32_bit_floats_are_refused():
  with pytest.raises(ValueError, match="magnitude"):
    ops.rotary(**rotary_args(magnitude=1e300))
  with pytest.raises(ValueError, match="eps"):
    ops.qk_norm_rotary(**rotary_args(), q_weight=None, k_weight=None, eps=1e300)


def test_more_heads_than_fit_are_refused():
  many = torch.zeros(1, 1, 8, dtype=BF).expand(1, (1 << 24) + 1, 8)
  with pytest.raises(ValueError, match="2\\^24"):
    ops.packed_attention(many, many, many, torch.tensor([0, 1], dtype=torch.int32))
  with pytest.raises(ValueError, match="2\\^24"):
    ops.rotary(many, None, torch.arange(1), ops.rotary_frequencies(8))


def rotary_args(**kw):
  a = dict(q=torch.zeros(5, 4, 32, dtype=BF), k=torch.zeros(5, 2, 32, dtype=BF), positions=torch.arange(5), freqs=ops.rotary_frequencies(32))
  a.update(kw)
  return a


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 32, dtype=BF)), r"\[..., H, D\]"),
    (dict(k=torch.zeros(4, 2, 32, dtype=BF)), r"\[..., H, D\]"),
    (dict(k=torch.zeros(5, 2, 16, dtype=BF)), r"\[..., H, D\]"),
    (dict(k=torch.zeros(5, 2, 32)), "alike"),
    (dict(q=torch.zeros(5, 4, 32, dtype=torch.float64), k=None), "bfloat16, float16 or float32"),
    (dict(q=torch.zeros(5, 1, 257, dtype=BF), k=None), r"1 .. 256"),
    (dict(q=torch.zeros(5, 0, 32, dtype=BF), k=None), "heads"),
    (dict(freqs=torch.zeros(8)), "float64"),
    (dict(freqs=torch.zeros(17, dtype=torch.float64)), "1 to 16"),
    (dict(freqs=torch.zeros(0, dtype=torch.float64)), "1 to 16"),
    (dict(positions=torch.zeros(5)), "int32 or int64"),
    (dict(positions=torch.arange(4)), "do not fit"),
    (dict(magnitude=math.inf), "magnitude"),
    (dict(out_q=torch.zeros(5, 4, 32)), "out_q must be"),
    (dict(k=None, out_k=torch.zeros(5, 2, 32, dtype=BF)), "out_k without k"),
])
def test_rotary_refuses(kw, match):
  with pytest.raises(ValueError, match=match):
    ops.rotary(**rotary_args(**kw))


def test_rotary_refuses_overlaps():
  x = torch.zeros(5, 6, 32, dtype=BF)
  q, k = x[:, :4], x[:, 4:]
  a = dict(positions=torch.arange(5), freqs=ops.rotary_frequencies(32))
  with pytest.raises(_Launched):
    ops.rotary(q, k, out_q=q, out_k=k, **a)
  for out_q, out_k in ((x[:, 1:5], None), (None, x[:, 3:5]), (x[:, 2:], k)):
    with pytest.raises(ValueError, match="overlap nothing else"):
      ops.rotary(q, k, out_q=out_q, out_k=out_k, **a)
  y = torch.zeros(5, 4, 32, dtype=BF)
  with pytest.raises(ValueError, match="overlap nothing else"):
    ops.rotary(y, y, out_q=y, **a)
  with pytest.raises(ValueError, match="overlap nothing else"):
    ops.rotary(q, q, out_q=y, out_k=y, **a)


@pytest.mark.parametrize("kw,match", [
    (dict(norm="batch"), "norm"),
    (dict(q_bias=torch.zeros(32)), "biases need"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"),
    (dict(q_weight=torch.zeros(16)), "weights and biases"),
    (dict(k=None), "without k"),
    (dict(q_weight=torch.zeros(32, requires_grad=True)), "no backward"),
])
def test_qk_norm_rotary_refuses(kw, match):
  a = dict(rotary_args(), q_weight=torch.ones(32), k_weight=torch.ones(32))
  a.update(kw)
  with pytest.raises(ValueError, match=match):
    ops.qk_norm_rotary(**a)


def c_error(lib, rc):
  assert rc != 0
  buf = C.create_string_buffer(1024)
  lib.sf_hip_last_error(buf, 1024)
  return buf.value.decode()


@pytest.fixture
def lib(monkeypatch):
  monkeypatch.undo()
  return _lib.load()


def packed_struct(**kw):
  cu = torch.zeros(3, dtype=torch.int32)
  a = _lib.PackedAttentionArgs(B=2, H=4, Hkv=2, D=32, Tq=6, Tk=6, scale=1.0, causal=0, dtype=0)
  for name in ("q", "k", "v", "out"):
    setattr(a, name, 4096)
  for name in ("q_s", "k_s", "v_s", "o_s"):
    getattr(a, name)[0], getattr(a, name)[1] = 128, 32
  a.cu_q = a.cu_k = cu.data_ptr()
  for name, value in kw.items():
    if name.endswith("_s"):
      getattr(a, name)[0], getattr(a, name)[1] = value
    else:
      setattr(a, name, value)
  return a


@pytest.mark.parametrize("kw,match", [
    (dict(B=0), "positive"), (dict(H=3), "evenly"), (dict(D=20), "multiple of 8"), (dict(D=136), "multiple of 8"),
    (dict(dtype=2), "element type"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(Tk=1 << 31), "exceed"), (dict(Tq=1 << 31), "exceed"), (dict(q=None), "non-null"), (dict(v=None), "non-null"),
    (dict(cu_k=None), "cu_q and cu_k"), (dict(k=4104), "aligned"), (dict(q_s=(100, 32)), "multiples of 8"),
    (dict(k_s=(24, 32)), "row strides"), (dict(v_s=(1 << 24, 32)), "row strides"), (dict(v_s=(0, 32)), "row strides"),
])
def test_c_attention_refuses(lib, kw, match):
  a = packed_struct(**kw)
  assert match in c_error(lib, lib.sf_hip_packed_attention_fwd(C.byref(a), None, 0, None))
  assert lib.sf_hip_packed_attention_workspace_bytes(C.byref(a)) == 0


def test_c_attention_workspace(lib):
  assert "null" in c_error(lib, lib.sf_hip_packed_attention_fwd(None, None, 0, None))
  a = packed_struct(B=1, Tq=1, Tk=8192)                        # one new token over many keys: sliced
  need = lib.sf_hip_packed_attention_workspace_bytes(C.byref(a))
  assert need > 0
  for ptr, n in ((None, need), (4096, need - 1), (4100, need)):
    assert "workspace" in c_error(lib, lib.sf_hip_packed_attention_fwd(C.byref(a), ptr, n, None))
  a = packed_struct(Tq=0, q=None, out=None)                    # nothing to do, nothing launched
  assert lib.sf_hip_packed_attention_fwd(C.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("B,Hkv,need", [(1, 8, None), (64, 8, None), (128, 32, None), (256, 32, 257 * 4), (1000, 1, 1001 * 4), (100000, 4, 100001 * 4)])
def test_c_attention_workspace_is_bounded(lib, B, Hkv, need):
  """One token a sequence over long caches: the slices' buffer, 256 MiB at most, or the tiles before each sequence."""
  a = packed_struct(B=B, H=2 * Hkv, Hkv=Hkv, D=128, Tq=B, Tk=B * 4096)
  got = lib.sf_hip_packed_attention_workspace_bytes(C.byref(a))
  assert got == need if need else 0 < got <= (256 << 20) + (1 << 16)


def test_c_rotary_refuses(lib):
  def struct(**kw):
    a = _lib.RotaryArgs(T=5, H=4, Hk=0, D=32, R=32, dtype=0, norm=0, magnitude=1.0)
    a.q = a.q_out = a.positions = a.freqs = 4096
    for name, value in kw.items():
      setattr(a, name, value)
    return a
  assert "null" in c_error(lib, lib.sf_hip_rotary_fwd(None, None))
  for kw, match in ((dict(T=-1), "sizes"), (dict(H=0), "sizes"), (dict(D=257), "sizes"), (dict(R=3), "rotated dims"), (dict(R=0), "rotated dims"),
                    (dict(R=34), "rotated dims"), (dict(dtype=7), "element type"), (dict(norm=3), "norm"), (dict(q=None), "non-null"),
                    (dict(Hk=2), "non-null"), (dict(freqs=None), "non-null")):
    assert match in c_error(lib, lib.sf_hip_rotary_fwd(C.byref(struct(**kw)), None))
  assert lib.sf_hip_rotary_fwd(C.byref(struct(T=0)), None) == 0


def test_rotary_frequencies():
  R, base = 64, 10000.0
  plain = [base ** (-2 * i / R) for i in range(R // 2)]
  near = lambda got, want: torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)
  assert near(ops.rotary_frequencies(R), plain)
  assert near(ops.rotary_frequencies(R, base=500.0), [500.0 ** (-2 * i / R) for i in range(R // 2)])
  assert near(ops.rotary_frequencies(R, scaling="linear", factor=4.0), [f / 4 for f in plain])
  stretched = ops.rotary_frequencies(R, scaling="base", factor=8.0)
  assert stretched[0] == 1.0 and abs(stretched[-1].item() - plain[-1] / 8) < 1e-13 * plain[-1]
  by_turns = ops.rotary_frequencies(R, scaling="turns", factor=8.0, original_length=4096, low_turns=1.0, high_turns=32.0)
  for f, got in zip(plain, by_turns.tolist()):
    turns = 4096 * f / (2 * math.pi)
    keep = min(max((turns - 1) / 31, 0), 1)
    assert abs(got - f * (keep + (1 - keep) / 8)) < 1e-13
  for kw in (dict(rotary_dim=5), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=-1.0),
             dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="turns"), dict(rotary_dim=2, scaling="base")):
    with pytest.raises(ValueError, match="rotary_frequencies"):
      ops.rotary_frequencies(**kw)


def tiles_bound(rows, B, R):
  return rows // R + min(B, rows)


@pytest.mark.parametrize("R", [32, 128])
def test_bound_of_the_row_tiles(R):
  """The launch has a workgroup for every row tile, wherever the sequences end."""
  g = torch.Generator().manual_seed(R)
  for B in (1, 2, 7, 63, 64, 65, 200):
    for top in (1, 2, 40, 500):
      lens = torch.randint(0, top + 1, (B,), generator=g).tolist()
      for G in (1, 3, 8):
        rows = sum(lens) * G
        assert sum(-(-n * G // R) for n in lens) <= tiles_bound(rows, B, R) or rows == 0


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 257, 4096, 4097, 20000])
def test_search_of_a_tile(B):
  """The search over the tiles before each sequence, 64 of them a step: the sequence that holds the tile."""
  g = torch.Generator().manual_seed(B)
  for top in (1, 4):
    tiles = torch.randint(0, top + 1, (B,), generator=g)
    starts = [0] + tiles.cumsum(0).tolist()
    for idx in range(0, starts[-1], 1 + starts[-1] // 500):
      b, n = 0, B
      while n > 1:
        step = -(-n // 64)
        at = [lane * step < n and starts[b + min(lane * step, n - 1)] <= idx for lane in range(64)]
        assert at == sorted(at, reverse=True)
        skip = max(sum(at) - 1, 0) * step
        b, n = b + skip, min(step, n - skip)
      assert starts[b] <= idx < starts[b + 1]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B", [2, 5, 20, 64])
def test_order_of_the_row_tiles(B, causal):
  """The search for the tile with the idx-th most keys: each tile once, keys falling in steps of 64."""
  g = torch.Generator().manual_seed(B)
  draw = lambda top: int(torch.randint(0, top, (1,), generator=g))
  for G, R in ((1, 128), (3, 128), (8, 256), (2, 32)):
    lk = [(0, 1, draw(900))[draw(3)] for _ in range(B)]
    lq = [(n, draw(600))[draw(2)] for n in lk]
    tiles = [-(-n * G // R) for n in lq]

    def longer(b, u):
      if u < 0:
        return tiles[b]
      if not causal:
        return tiles[b] if lk[b] > 64 * u else 0
      token = 64 * u - (lk[b] - lq[b])
      return tiles[b] if token <= 0 else 0 if token >= lq[b] else tiles[b] - token * G // R

    def keys(b, t):
      return max(0, (min((t + 1) * R, lq[b] * G) - 1) // G + lk[b] - lq[b] + 1) if causal else lk[b]

    order = []
    for idx in range(sum(tiles)):
      step, u = 1, -1
      while any(n > 64 * step for n in lk):
        step *= 2
      while step > 0:
        u += step if sum(longer(b, u + step) for b in range(B)) > idx else 0
        step //= 2
      above = [longer(b, u + 1) for b in range(B)]
      rank, b = idx - sum(above), 0
      while rank >= longer(b, u) - above[b]:
        rank -= longer(b, u) - above[b]
        b += 1
      order.append((b, tiles[b] - 1 - above[b] - rank))
    assert sorted(order) == [(b, t) for b in range(B) for t in range(tiles[b])]
    steps = [-(-keys(b, t) // 64) for b, t in order]
    assert steps == sorted(steps, reverse=True)


@pytest.mark.parametrize("share", [1, 16, 32, 128, 256])
def test_key_slices_of_different_sequences(share):
  """Slices dealt out by keys: every tile has its own, no more than the launch, and tiles that do not exist are noted so."""
  g = torch.Generator().manual_seed(share)
  draw = lambda top: int(torch.randint(0, top, (1,), generator=g))
  ceil = lambda a, b: -(-a // b)
  for trial in range(40):
    B, unit = 1 + draw(64), (128, 256)[draw(2)]
    tiles = [draw(3) for _ in range(B)]
    units = [ceil((0, 1, draw(300), draw(70000))[draw(4)], unit) for _ in range(B)]
    bound, all_tiles = sum(tiles) + draw(5), sum(tiles)
    total = sum(n * u for n, u in zip(tiles, units))
    assert total < 1 << 23
    over = lambda n: max(ceil(total, n), 1)
    split = lambda c: [max(ceil(u, c), 1) for u in units]
    used = lambda c: sum(n * z for n, z in zip(tiles, split(c)))
    c = over(share)
    high = c if share <= all_tiles or used(c) <= share else over(share - all_tiles)
    while c < high:
      mid = (c + high) // 2
      c, high = (c, mid) if used(mid) <= share else (mid + 1, high)
    z = split(c)
    assert used(c) <= share + all_tiles and (share <= all_tiles or used(c) <= share)
    noted, slices = set(), []
    for item in range(share + bound):
      b, before, slot = 0, 0, 0
      while b < B and item >= before + tiles[b] * z[b]:
        before, slot, b = before + tiles[b] * z[b], slot + tiles[b], b + 1
      if b == B:
        slot = all_tiles + item - before
        if slot < bound:
          assert slot not in noted
          noted.add(slot)
        continue
      tile, slice_ = divmod(item - before, z[b])
      slices.append((b, tile, slice_))
      if slice_ == 0:
        assert slot + tile not in noted
        noted.add(slot + tile)
    assert noted == set(range(bound))
    assert slices == [(b, t, i) for b in range(B) for t in range(tiles[b]) for i in range(z[b])]


@pytest.mark.parametrize("name", ["sf_packed_attention_args", "sf_rotary_args"])
def test_filled_structs(name):
  """The packed fields are the constructor's."""
  struct = _lib.STRUCTS[name]
  fill = {"sf_packed_attention_args": _lib.packed_attention_args, "sf_rotary_args": _lib.rotary_args}[name]
  values, flat = [], []
  for i, (_, t) in enumerate(struct._fields_):
    if issubclass(t, C.Array):
      values.append((-i, 1 << 40))
      flat += [-i, 1 << 40]
    else:
      values.append(i / 4 if t is C.c_float else None if t is C.c_void_p and i % 2 else i)
      flat.append(values[-1] or 0)
  a, b = struct(*values), fill(*flat)
  for field, t in struct._fields_:
    x, y = getattr(a, field), getattr(b, field)
    assert list(x) == list(y) if issubclass(t, C.Array) else x == y
  with pytest.raises(Exception, match="argument out of range|format requires"):
    fill(*([1 << 40] * len(flat)))
