"""The paged cache of keys and values: new rows into their pages, and attention over them against its definition in
64 bits, with the tolerance of the attention over packed sequences (its derivation stands there)."""
import math

import pytest
import torch

from sparsefold_amd.backends.hip import ops
from test_gpu_packed_attention import DEV, TYPES, check, definition, offsets

pytestmark = pytest.mark.gpu


def paged(k, v, lens, rows, layout="rows", spare=3, seed=0, fill=math.nan, width=None):
  """Pages of ``rows`` rows in random order that hold the sequences' keys laid end to end in k and v; free rows and pages
  hold ``fill``; behind a sequence's pages the table names pages that do not exist."""
  g = torch.Generator().manual_seed(seed)
  H, D = k.shape[1:]
  need = [-(-n // rows) for n in lens]
  P = sum(need) + spare
  order = torch.randperm(P, generator=g)
  table = torch.full((len(lens), max(max(need), 1) if width is None else width), 1 << 30, dtype=torch.int32)
  shape = {"rows": (P, rows, H, D), "heads": (P, H, rows, D), "both": (P, 2, rows, H, D), "wide": (P, rows, H, D + 24)}[layout]
  kc, vc = (torch.full(shape, fill, dtype=k.dtype, device=DEV) for _ in range(2))
  if layout == "heads":
    kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
  elif layout == "both":
    kc, vc = kc[:, 0], kc[:, 1]
  elif layout == "wide":
    kc, vc = kc[..., 8:8 + D], vc[..., 16:16 + D]
  at = page = 0
  for b, n in enumerate(lens):
    for i in range(need[b]):
      p, m = int(order[page]), min(rows, n - i * rows)
      table[b, i] = p
      kc[p, :m], vc[p, :m] = k[at:at + m], v[at:at + m]
      at, page = at + m, page + 1
  return kc, vc, table.to(DEV)


def make(lens_q, lens_k, H, Hk, D, dtype, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda t, h: torch.randn(t, h, D, generator=g).to(dtype).to(DEV)
  return r(sum(lens_q), H), r(sum(lens_k), Hk), r(sum(lens_k), Hk)


def ints(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


def run(lens_q, lens_k, H, Hk, D, dtype, rows, causal=True, layout="rows", seed=0, **kw):
  q, k, v = make(lens_q, lens_k, H, Hk, D, dtype, seed)
  kc, vc, table = paged(k, v, lens_k, rows, layout, seed=seed)
  out = ops.paged_attention(q, kc, vc, table, offsets(lens_q), ints(lens_k), causal=causal, **kw)
  check(out, q, k, v, lens_q, lens_k, causal)
  return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [([1, 1, 1], [70, 1, 333]), ([70, 1, 33], [170, 1, 100]), ([150, 90], [333, 90])], ids=str)
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128])
def test_head_dims(D, lens, dtype):
  run(*lens, 4, 2, D, TYPES[dtype], 16, seed=D)


@pytest.mark.parametrize("rows", [16, 32, 48, 64, 80, 112, 128, 1008, 4096])
@pytest.mark.parametrize("lens", [([1] * 5, [15, 16, 17, 1000, 4097]), ([200, 1, 31], [300, 64, 2000]), ([9], [3000])], ids=lambda l: str(sum(l[0])))
def test_page_sizes(rows, lens):
  run(*lens, 8, 2, 64, torch.bfloat16, rows, seed=rows)
  run(*lens, 4, 2, 128, torch.float16, rows, seed=rows)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (6, 2), (8, 8), (5, 1), (33, 1), (40, 8)])
def test_head_groups(heads, causal):
  run([130, 64, 5, 1], [330, 64, 5, 200], *heads, 64, torch.bfloat16, 32, causal, seed=heads[0])


LENGTHS = [([1], [1]), ([2], [1]), ([0, 3, 0], [4, 0, 0]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [127, 128, 129]),
           ([255, 257], [256, 255]), ([1, 1, 1, 1], [1, 65, 1000, 0]), ([5], [700]), ([700], [5]), ([300, 2], [1100, 3]),
           ([1] * 70, [(7 * i) % 90 for i in range(70)]), ([1] * 300, [(11 * i) % 200 for i in range(300)]),
           ([3] * 250, [(5 * i) % 64 for i in range(250)])]


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("bf16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS, ids=lambda l: "x".join(str(sum(x)) for x in l))
def test_lengths(lens, causal, dtype, D):
  run(*lens, 4, 2, D, TYPES[dtype], 16, causal, seed=5)


@pytest.mark.parametrize("dtype,D,n,m", [("bf16", 128, 1, 9001), ("fp16", 64, 3, 5000), ("bf16", 48, 2, 3300), ("bf16", 96, 1, 2050),
                                         ("bf16", 128, 200, 6000), ("fp16", 32, 333, 4097), ("bf16", 80, 600, 5000)])
def test_key_slices(dtype, D, n, m):
  """Few rows and many keys: workgroups take slices of the keys; the sums have one order."""
  one = run([n], [m], 8, 2, D, TYPES[dtype], 16, seed=m)
  assert torch.equal(one, run([n], [m], 8, 2, D, TYPES[dtype], 16, seed=m))


@pytest.mark.parametrize("lens_q,lens_k", [([1] * 32, [8192 // (1 + i) for i in range(32)]), ([512] + [1] * 6, [3000, 5, 700, 1, 2500, 64, 900])], ids=["tokens", "mixed"])
@pytest.mark.parametrize("max_len", [None, 1, 300, 1 << 40])
def test_the_launch_is_chosen_by_max_len_but_no_result(lens_q, lens_k, max_len):
  run(lens_q, lens_k, 16, 4, 128, torch.bfloat16, 64, seed=3, max_len=max_len)


def test_long_piece_takes_the_widest_tiles():
  """Rows enough for tiles of 256; sampled rows."""
  n, m, H, Hk, D = 4096, 5000, 32, 8, 128
  q, k, v = make([n], [m], H, Hk, D, torch.bfloat16, 2)
  kc, vc, table = paged(k, v, [m], 16)
  out = ops.paged_attention(q, kc, vc, table, offsets([n]), ints([m]))
  assert torch.isfinite(out.float()).all()
  for r in (0, 1, 63, 255, 256, 1000, 2049, 4000, 4095):
    seen = m - n + r + 1
    want, tol = definition(q[r:r + 1], k[:seen], v[:seen], False, 1 / math.sqrt(D))
    assert ((out[r:r + 1].cpu().double() - want).abs() <= tol).all(), r


@pytest.mark.parametrize("layout", ["rows", "heads", "both", "wide"])
@pytest.mark.parametrize("lens", [([1, 1], [1000, 77]), ([140, 3], [500, 3])], ids=str)
def test_layouts_of_the_pages(layout, lens):
  run(*lens, 6, 3, 64, torch.bfloat16, 32, layout=layout)
  run(*lens, 6, 3, 72, torch.float16, 48, layout=layout)


@pytest.mark.parametrize("lens_q,lens_k", [([1, 1, 1], [100, 37, 64]), ([150, 2], [333, 40])], ids=str)
def test_strided_queries_table_and_out(lens_q, lens_k):
  q, k, v = make(lens_q, lens_k, 4, 2, 64, torch.bfloat16, 1)
  kc, vc, table = paged(k, v, lens_k, 16)
  B = len(lens_q)
  want = ops.paged_attention(q, kc, vc, table, offsets(lens_q), ints(lens_k))
  wide = torch.full((B, table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
  wide[:, :table.shape[1]] = table
  fused = torch.zeros(q.shape[0], 9, 64, dtype=q.dtype, device=DEV)
  fused[:, 2:6] = q
  room = torch.zeros(q.shape[0], 7, 64, dtype=q.dtype, device=DEV)
  got = ops.paged_attention(fused[:, 2:6], kc, vc, wide[:, :table.shape[1]], offsets(lens_q), ints(lens_k), out=room[:, 1:5])
  assert torch.equal(got, want) and (room[:, 0] == 0).all() and (room[:, 5:] == 0).all()
  odd = torch.zeros(q.shape[0] * 4 * 64 + 3, dtype=q.dtype, device=DEV)[3:].view(q.shape)     # rows that are not aligned are copied
  odd.copy_(q)
  assert torch.equal(ops.paged_attention(odd, kc, vc, table.t().contiguous().t(), offsets(lens_q), ints(lens_k)), want)


def test_padded_queries_and_rows_outside_stay():
  q, k, v = make([8, 8, 8], [50, 9, 300], 4, 2, 32, torch.float16, 4)
  kc, vc, table = paged(k, v, [50, 9, 300], 16)
  out = torch.full_like(q, 7.0)
  ops.paged_attention(q[:22], kc, vc, table, ints([0, 8, 16, 22]), ints([50, 9, 300]), len_q=ints([3, 0, 6]), out=out[:22])
  starts = [(0, 3, 0, 50), (16, 6, 59, 300)]
  for at, n, ak, m in starts:
    want, tol = definition(q[at:at + n], k[ak:ak + m], v[ak:ak + m], True, 1 / math.sqrt(32))
    assert ((out[at:at + n].cpu().double() - want).abs() <= tol).all()
  for a, b in ((3, 8), (8, 16), (22, 24)):
    assert (out[a:b] == 7.0).all()


@pytest.mark.parametrize("n", [1, 5, 200])
def test_lengths_past_the_table_and_pages_outside_the_cache(n):
  """Lengths are clamped to the table's pages; pages that do not exist count as zeros."""
  m, D = 320, 64
  q, k, v = make([n], [m], 4, 2, D, torch.bfloat16, n)
  kc, vc, table = paged(k, v, [m], 64)
  out = ops.paged_attention(q, kc, vc, table, offsets([n]), ints([10 * m]))
  check(out, q, k, v, [n], [m], True)
  for bad in (-1, kc.shape[0], 1 << 30):
    t = table.clone()
    t[0, 1] = bad
    k2, v2 = k.clone(), v.clone()
    k2[64:128], v2[64:128] = 0, 0
    check(ops.paged_attention(q, kc, vc, t, offsets([n]), ints([m])), q, k2, v2, [n], [m], True)
  zero = ops.paged_attention(q, kc, vc, table, offsets([n]), ints([-5]))
  assert (zero == 0).all()


@pytest.mark.parametrize("n", [1, 3, 150])
def test_shared_pages(n):
  """Two sequences of one beginning name the same pages."""
  q, k, v = make([n, n], [400, 60], 4, 2, 64, torch.bfloat16, 9)
  kc, vc, table = paged(k, v, [400, 60], 16)
  table[1, 4:10] = table[1, :6].clone()
  table[1, :4] = table[0, :4]
  lens = [400, 64 + 60]
  out = ops.paged_attention(q, kc, vc, table, offsets([n, n]), ints(lens))
  kk, vv = (torch.cat((x[:400], x[:64], x[400:])) for x in (k, v))
  check(out, q, kk, vv, [n, n], lens, True)


@pytest.mark.parametrize("n,D", [(1, 64), (4, 128), (200, 64), (300, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_later_keys_have_no_influence(n, D, bad):
  m = n + 200
  q, k, v = make([n], [m], 4, 2, D, torch.bfloat16, n)
  kc, vc, table = paged(k, v, [m], 16)
  want = ops.paged_attention(q, kc, vc, table, offsets([n]), ints([m]))
  last = m - 1
  p, r = int(table[0, last // 16]), last % 16
  kc[p, r], vc[p, r] = bad, bad
  got = ops.paged_attention(q, kc, vc, table, offsets([n]), ints([m]))
  check(got[:n - 1], q[:n - 1], k[:last], v[:last], [n - 1], [last], True)
  if n > 1:
    assert torch.isfinite(want).all()


def test_cache_past_32_bits():
  """Pages that lie more than 2^32 bytes apart, the last ones in use."""
  P, R, Hk, D = (1 << 31) // (64 * 8 * 128) + 40, 64, 8, 128
  kc = torch.zeros(P, R, Hk, D, dtype=torch.bfloat16, device=DEV)
  vc = torch.zeros(P, R, Hk, D, dtype=torch.bfloat16, device=DEV)
  k, v = torch.randn(400, Hk, D, device=DEV).to(kc.dtype), torch.randn(400, Hk, D, device=DEV).to(kc.dtype)
  table = ints([[P - 1, 0, P - 5, 3, P - 2, P // 2, 7]])
  ops.paged_cache_write(k, v, kc, vc, table, offsets([400]), ints([400]))
  for i, p in enumerate(table[0].tolist()):
    n = min(64, 400 - 64 * i)
    assert torch.equal(kc[p, :n], k[64 * i:64 * i + n]) and torch.equal(vc[p, :n], v[64 * i:64 * i + n])
  for n in (1, 100):
    q = torch.randn(n, 8, D, device=DEV).to(kc.dtype)
    check(ops.paged_attention(q, kc, vc, table, offsets([n]), ints([400])), q, k, v, [n], [400], True)


# ---- writes ---------------------------------------------------------------------------

def written(k, v, kc, vc, table, lens, lens_k):
  """The pages after the write, one row after another."""
  kc, vc, rows, at = kc.clone(), vc.clone(), kc.shape[1], 0
  for b, n in enumerate(lens):
    for i in range(n):
      j = lens_k[b] - n + i
      if 0 <= j < table.shape[1] * rows and 0 <= int(table[b, j // rows]) < kc.shape[0]:
        kc[int(table[b, j // rows]), j % rows], vc[int(table[b, j // rows]), j % rows] = k[at + i], v[at + i]
    at += n
  return kc, vc


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("layout", ["rows", "heads", "both", "wide"])
@pytest.mark.parametrize("heads,D,rows", [(1, 8, 16), (2, 64, 16), (8, 128, 64), (3, 40, 48), (5, 24, 32), (1, 128, 16)])
def test_write(heads, D, rows, layout, dtype):
  lens, lens_k = [1, 0, 37, 5, 70, 1], [1, 9, 50, 64, 70, 200]
  _, k, v = make([0], lens_k, 1, heads, D, TYPES[dtype], D)
  kc, vc, table = paged(k, v, lens_k, rows, layout, fill=3.0)
  new = torch.randn(sum(lens), 2 * heads, D, device=DEV).to(k.dtype)
  want = written(new[:, :heads], new[:, heads:], kc, vc, table, lens, lens_k)
  ops.paged_cache_write(new[:, :heads], new[:, heads:], kc, vc, table, offsets(lens), ints(lens_k))
  assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


@pytest.mark.parametrize("B", [1, 63, 64, 65, 130, 5000])
def test_write_finds_its_sequence_among_many(B):
  g = torch.Generator().manual_seed(B)
  lens = [int(x) for x in torch.randint(0, 3, (B,), generator=g)]
  lens_k = [n + int(x) for n, x in zip(lens, torch.randint(0, 14, (B,), generator=g))]
  kc, vc = (torch.zeros(B, 16, 1, 8, dtype=torch.bfloat16, device=DEV) for _ in range(2))
  table = torch.randperm(B, generator=g).to(torch.int32)[:, None]
  k, v = torch.randn(sum(lens), 1, 8).bfloat16(), torch.randn(sum(lens), 1, 8).bfloat16()
  want = written(k, v, kc.cpu(), vc.cpu(), table, lens, lens_k)
  ops.paged_cache_write(k.to(DEV), v.to(DEV), kc, vc, table.to(DEV), offsets(lens), ints(lens_k))
  assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


def test_write_drops_what_has_no_place():
  """Places before 0, past the table, and pages outside the cache; a padded batch."""
  k, v = torch.randn(40, 2, 16, device=DEV).half(), torch.randn(40, 2, 16, device=DEV).half()
  kc, vc = (torch.zeros(4, 16, 2, 16, dtype=torch.float16, device=DEV) for _ in range(2))
  table = ints([[0, -1], [1, 4], [2, 1 << 30], [3, 3]])
  lens_k = [20, 3, 100, 32]
  want = written(k, v, kc.cpu(), vc.cpu(), table.cpu(), [10, 10, 10, 0], lens_k)
  ops.paged_cache_write(k, v, kc, vc, table, ints([0, 10, 20, 30, 40]), ints(lens_k), len_new=ints([10, 10, 10, 0]))
  assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
  ops.paged_cache_write(k, v, kc, vc, table, ints([0, 10, 20, 30, 40]), ints([5, 5, 5, 5]), len_new=ints([5, 2, 0, 0]))
  assert torch.equal(kc[0, :5], k[:5]) and torch.equal(kc[1, 3:5], k[10:12]) and torch.equal(vc[0, :5], v[:5])
  before = kc.clone()
  ops.paged_cache_write(k, v, kc, vc, table, ints([-3, 50, 20, 7, 1 << 30]), ints([-4, 0, -1, 0]))    # offsets that fall: nothing outside is written
  assert torch.equal(before, kc)


def test_write_of_nothing():
  k = torch.zeros(0, 2, 16, dtype=torch.bfloat16, device=DEV)
  kc, vc = (torch.ones(2, 16, 2, 16, dtype=torch.bfloat16, device=DEV) for _ in range(2))
  ops.paged_cache_write(k, k, kc, vc, ints([[0]]), ints([0, 0]), ints([0]))
  assert (kc == 1).all()
  assert ops.paged_attention(torch.zeros(0, 4, 16, dtype=torch.bfloat16, device=DEV), kc, vc, ints([[0]]), ints([0, 0]), ints([0])).shape == (0, 4, 16)


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [128, 60, 1, 11]], ids=str)
def test_capture_and_replay(lens):
  """A captured step of write and attention follows the lengths, the table and the rows at each replay; two graphs at once."""
  H, Hk, D, R = 8, 2, 128, 16
  g = torch.Generator().manual_seed(1)
  T = sum(lens)
  q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hk, Hk))
  kc, vc = (torch.randn(400, R, Hk, D, generator=g).bfloat16().to(DEV) for _ in range(2))
  table = torch.randperm(400, generator=g)[:320].view(4, 80).to(torch.int32).to(DEV)
  cu, lk = offsets(lens), ints([900, 300, 77, 11])

  def step():
    ops.paged_cache_write(k, v, kc, vc, table, cu, lk)
    return ops.paged_attention(q, kc, vc, table, cu, lk)

  step()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  graphs, outs = [], []
  with torch.cuda.stream(side):
    for _ in range(2):
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph, stream=side):
        outs.append(step())
      graphs.append(graph)
  for i in range(4):
    for t in (q, k, v):
      t.copy_(torch.randn_like(t))
    lk.copy_(ints([[900, 300, 77, 11], [1, 1, 1, 1], [1280, 512, 600, 200], [128, 60, 1, 0]][i]))
    table.copy_(table[:, torch.randperm(80)])
    graphs[i % 2].replay()
    torch.cuda.synchronize()
    got = outs[i % 2].clone()
    assert torch.equal(got, step())


def test_other_streams_at_once():
  """Calls on two streams, each with its own workspace, give what they give alone."""
  sets = []
  for seed in (1, 2):
    q, k, v = make([1] * 4, [4000, 100, 2000, 3000], 8, 2, 128, torch.bfloat16, seed)
    sets.append((q, *paged(k, v, [4000, 100, 2000, 3000], 16, seed=seed)))
  cu, lk = offsets([1] * 4), ints([4000, 100, 2000, 3000])
  want = [ops.paged_attention(*s, cu, lk) for s in sets]
  streams = [torch.cuda.Stream() for _ in sets]
  torch.cuda.synchronize()
  got = [None, None]
  for _ in range(10):
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        got[i] = ops.paged_attention(*sets[i], cu, lk)
  torch.cuda.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_agrees_with_the_packed_attention():
  """Over the same keys the two kernels differ by the order of their sums at most."""
  lens_q, lens_k = [100, 1, 300], [400, 900, 300]
  q, k, v = make(lens_q, lens_k, 8, 2, 96, torch.bfloat16, 8)
  kc, vc, table = paged(k, v, lens_k, 64)
  a = ops.paged_attention(q, kc, vc, table, offsets(lens_q), ints(lens_k))
  b = ops.packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=True)
  at = ak = 0
  for n, m in zip(lens_q, lens_k):
    _, tol = definition(q[at:at + n], k[ak:ak + m], v[ak:ak + m], True, 1 / math.sqrt(96))
    assert ((a[at:at + n] - b[at:at + n]).cpu().double().abs() <= 2 * tol).all()
    at, ak = at + n, ak + m


def test_write_of_more_tokens_than_a_launch_dimension_holds():
  """2^26 tokens, a wave each: 2^24 workgroups of 256 threads and some.  The pages of the first tokens, of those on both sides of each grid
  row's border and of the last are in the cache; the others are dropped."""
  T, Hk, D, R = (1 << 26) + 5, 5, 128, 64
  rows = torch.empty((T + 1) * 8 + Hk * D, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(4))
  k, v = (rows.as_strided((T, Hk, D), (8, D, 1), at) for at in (0, 8))                # (rows that overlap)
  used = sorted({0} | {p for b in range(1, 5) for p in ((b << 24) // R - 1, (b << 24) // R)} | {T // R})
  table = torch.full((1, T // R + 1), -1, dtype=torch.int32, device=DEV)
  table[0, used] = torch.arange(len(used), dtype=torch.int32, device=DEV)
  kc, vc = (torch.full((len(used) + 1, R, Hk, D), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
  ops.paged_cache_write(k, v, kc, vc, table, ints([0, T]), ints([T]))
  for i, p in enumerate(used):
    n = min(R, T - p * R)
    for cache, new in ((kc, k), (vc, v)):
      assert torch.equal(cache[i, :n], new[p * R:p * R + n]) and (cache[i, n:] == 3).all()
  assert (kc[-1] == 3).all() and (vc[-1] == 3).all()


@pytest.mark.parametrize("heads,D,rows", [(1, 8, 16), (1, 32, 48), (3, 40, 16), (2, 64, 32), (5, 48, 16), (8, 64, 16)])
@pytest.mark.parametrize("T", [8192, 8193, 30000])
def test_write_of_narrow_rows(T, heads, D, rows):
  """Numbers of tokens on both sides of where a wave takes several rows; sequences of no and of one new token among others, and
  tokens without a place."""
  g = torch.Generator().manual_seed(T + D)
  cut = torch.sort(torch.randint(0, T + 1, (99,), generator=g)).values.tolist()
  lens = [b - a for a, b in zip([0, *cut, cut[-1] + 1], [*cut, cut[-1] + 1, T])] if cut[-1] < T else [b - a for a, b in zip([0, *cut], [*cut, T])]
  lens_k = [n + int(x) for n, x in zip(lens, torch.randint(0, 50, (len(lens),), generator=g))]
  need = [-(-n // rows) for n in lens_k]
  P, order = sum(need), torch.randperm(sum(need), generator=g).to(torch.int32)
  table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
  at = 0
  for b, n in enumerate(need):
    table[b, :n] = order[at:at + n]
    at += n
  table[7, 0] = P                                              # (a page outside the cache)
  k, v = (torch.randn(T, heads, D, generator=g).bfloat16() for _ in range(2))
  kc, vc = (torch.zeros(P, rows, heads, D, dtype=torch.bfloat16) for _ in range(2))
  b = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
  place = torch.tensor(lens_k)[b] - torch.tensor(lens)[b] + torch.arange(T) - torch.tensor([0, *lens]).cumsum(0)[b]
  page = table[b, place // rows].long()
  there = (page >= 0) & (page < P)
  want = kc.clone(), vc.clone()
  for w, new in zip(want, (k, v)):
    w[page[there], (place % rows)[there]] = new[there]
  kc, vc = kc.to(DEV), vc.to(DEV)
  ops.paged_cache_write(k.to(DEV), v.to(DEV), kc, vc, table.to(DEV), offsets(lens), ints(lens_k))
  assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
