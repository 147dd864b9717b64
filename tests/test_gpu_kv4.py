"""The paged 4-bit cache against 64 bits: rows written and read, attention of single tokens and of prompts, pages."""
import itertools
import random

import numpy as np
import pytest
import torch

import _kv4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _angles(n, rd=64):
    f = 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _rows(g, n, d):
    x = torch.randn(n, d, generator=g) * 0.5
    x[:, :: max(1, d // 9)] *= 6
    return x.to(BF)


def _filled(g, counts, dim, page, spare=3):
    """A cache whose sequence s holds counts[s] random rows in scattered pages, and its rows in 64 bits (on the grid)."""
    from dsv41_amd.kv4 import PagedKV4
    need = [-(-n // page) for n in counts]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(counts), max(max(need), 1) + 1), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    pool = torch.zeros(pages, page, R.ROW_BYTES[dim], dtype=torch.uint8)
    rows, at = [], 0
    for s, n in enumerate(counts):
        mine = order[at:at + need[s]]
        at += need[s]
        table[s, :need[s]] = mine.to(torch.int32)
        refs[mine] = 1
        x = _rows(g, n, dim)
        packed = torch.zeros(need[s] * page, R.ROW_BYTES[dim], dtype=torch.uint8)
        if n:
            packed[:n] = R.pack(x.double())
        pool[mine] = packed.view(need[s], page, R.ROW_BYTES[dim])
        rows.append(R.grid(x.double())[0] if n else torch.zeros(0, dim, dtype=torch.float64))
    return PagedKV4(pool.to(DEV), table.to(DEV), refs.to(DEV), dim=dim), rows


def _close(o, ref, rows_abs):
    """fp32 sums of fp16 probabilities (2^-12 of each term: 2^-11 of the largest value, sums of hundreds of terms far
    below) and one rounding to bf16 (2^-8 of the value at most half of that); window rows' probabilities are bf16 (2^-9 of
    each term), so 2^-8 of the largest value bounds what a sum of them is off by."""
    o = o.double().cpu()
    assert torch.equal(torch.isnan(o), torch.isnan(ref))
    o, ref = o.nan_to_num(0.0), ref.nan_to_num(0.0)
    err = (o - ref).abs()
    bound = ref.abs() * 2.0 ** -8 + rows_abs * 2.0 ** -8
    assert bool((err <= bound).all()), f"max {err.max().item():.3e}, bound there {bound.flatten()[err.argmax()].item():.3e}"
    assert err.norm() <= 2.0 ** -8 * ref.norm() + 1e-30  # (as a whole: a rounding of half that)


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("dim", [512, 576])
@pytest.mark.parametrize("page,start,n", [(16, 0, 1), (16, 15, 3), (64, 0, 64), (64, 63, 130), (256, 7, 300)])
def test_append_and_read(dim, page, start, n):
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(n + dim)
    c = PagedKV4.empty(9 + 2 * (start + n) // page, 3, start + n + 5, dim, page, DEV)
    c.reserve([2, 0], [0, 0], [start + n, start + n])
    x = _rows(g, 2 * n, dim)
    cos, sin = _angles((start + n) * 4)
    seq = torch.tensor([2] * n + [0] * n)
    row = torch.arange(start, start + n).repeat(2)
    row[n // 2] = -1
    c.append(x.to(DEV), seq, row, 4, cos.to(DEV), sin.to(DEV), 64)
    got = c.read(seq, row)
    y = R.rotate(x.double(), cos, sin, row.clamp_min(0) * 4, 64).to(BF).double()
    want, _, _ = R.grid(y)
    want[row < 0] = 0
    assert got.shape == (2 * n, dim) and torch.equal(got.double().cpu(), want)
    # the bytes, and nothing beside them
    packed = R.pack(y)
    flat, pool = torch.zeros_like(c.pool).cpu(), c.pool.cpu()
    table = c.table.cpu()
    for i in range(2 * n):
        if row[i] >= 0:
            flat[table[seq[i], row[i] // page], row[i] % page] = packed[i]
    assert torch.equal(pool, flat)
    c.check()


def test_append_matches_the_bf16_cache():
    """The rows that cache.append_compressed_decode stores in bf16: the same but where fp32 and 64 bits round a rotated
    value to another bf16 (2^-16 of them) that lies on another side of the grid's border."""
    from dsv41_amd import cache as C
    from dsv41_amd.kv4 import PagedKV4
    g, n, dim = _gen(5), 700, 512
    x = _rows(g, n, dim).to(DEV)
    cos, sin = (t.to(DEV) for t in _angles(n * 4))
    tab = torch.zeros(1, n, dim, dtype=BF, device=DEV)
    row = torch.arange(n, device=DEV)
    C.append_compressed_decode(tab, x, (row + 1) * 4 - 1, torch.zeros(n, dtype=torch.int64, device=DEV), row, 4, cos, sin, 64)
    c = PagedKV4.empty(11, 1, n, dim, 64, DEV)
    c.reserve([0], [0], [n])
    c.append(x, [0] * n, row, 4, cos, sin, 64)
    got = c.read(torch.zeros(n, dtype=torch.int64), row)
    assert (got != tab[0]).any(1).sum().item() <= 2
    assert torch.equal(got[:, :448], tab[0, :, :448])


@pytest.mark.parametrize("dim", [512, 576])
def test_append_far_values(dim):
    """Ties, zeros, the smallest scales, saturation, infinities and NaN, in both parts of a row."""
    from dsv41_amd.kv4 import PagedKV4
    vals = [0.0, -0.0, 2.0 ** -12, 2.0 ** -9 * 6, 2.0 ** -9 * 9, 1.0, 2.5, 3.5, 5.0, 0.25, 0.75, 6.0, 100.0, 2688.0, 3000.0,
            1e30, float("inf"), float("nan"), -float("inf"), 3.3e38]
    g = _gen(1)
    x = torch.zeros(len(vals) + 1, dim, dtype=BF)
    for i, v in enumerate(vals):
        x[i] = torch.randn(dim, generator=g).to(BF) * 2
        x[i, 3::32] = v
        x[i, -7] = v
    x[-1] = torch.tensor([(-1) ** k * k / 4 for k in range(dim)]).clamp(-6, 6)
    n = len(x)
    c = PagedKV4.empty(2, 1, n, dim, 64, DEV)
    c.reserve([0], [0], [n])
    c.append(x.to(DEV), [0] * n, list(range(n)), 1, None, None, 0)
    got, want = c.read([0] * n, list(range(n))).double().cpu(), R.grid(x.double())[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_append_drops_and_notes():
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(4, 3, 64, 512, 16, DEV)
    c.reserve([0], [0], [20])
    c.fork([0], [1])
    before = c.pool.clone()
    x = torch.ones(6, 512, dtype=BF, device=DEV)
    cos, sin = (t.to(DEV) for t in _angles(40))
    # shared, no page, beyond the table, no such sequence, no angle (row 19 * 4), none
    c.append(x, [1, 0, 2, 7, 0, 0], [3, 40, 9000, 0, 19, -1], 4, cos, sin, 64)
    assert torch.equal(c.pool, before)
    with pytest.raises(RuntimeError, match="left out.*dropped"):
        c.check()
    c.check()
    assert not c.read([9, 0, 0, -1], [0, 63, 1 << 40, 3]).any()


@pytest.mark.parametrize("ratio", [1, 2, 4, 128])
def test_append_decode(ratio):
    """The rows by the tokens' positions: those that close a group, the first and the last of a page among them."""
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(ratio)
    pos = torch.tensor([0, ratio - 1, 17 * ratio - 1, 17 * ratio, 16 * ratio - 1, 32 * ratio - 2, 32 * ratio - 1, -1, 1 << 40])
    seq = torch.arange(9)
    x = _rows(g, 9, 576).to(DEV)
    cos, sin = (t.to(DEV) for t in _angles(33 * ratio))
    a, b = (PagedKV4.empty(30, 9, 40, 576, 16, DEV) for _ in range(2))
    for c in (a, b):
        c.reserve(seq, [0] * 9, [40] * 9)
    a.append_decode(x, seq, pos, ratio, cos, sin, 64)
    row = [int(p + 1) // ratio - 1 if p >= 0 and p < 1 << 31 and (p + 1) % ratio == 0 else -1 for p in pos]
    b.append(x, seq, row, ratio, cos, sin, 64)
    a.check()
    assert torch.equal(a.pool, b.pool) and sum(r >= 0 for r in row) >= 4


def test_index_arguments(monkeypatch):
    """Lists and tensors of any integer type are the same; others, and host memory in a capture, are refused; the tensors of
    a cache stay."""
    from dsv41_amd.kv4 import PagedKV4, sparse_attn4
    c = PagedKV4.empty(4, 2, 40, 512, 16, DEV)
    c.reserve([0, 1], torch.tensor([0, 0], dtype=torch.int32), torch.tensor([20, 3], dtype=torch.int16, device=DEV))
    c.append(torch.full((2, 512), 6.0, dtype=BF, device=DEV), torch.tensor([0, 9, 1, 9], device=DEV)[::2], [19, 2], 4, None, None, 0)
    c.check()
    assert c.read([0, 1], torch.tensor([19, 2], dtype=torch.uint8)).eq(6).all() and c.read([], []).shape == (0, 512)
    q, sink = torch.zeros(1, 1, 16, 512, dtype=BF, device=DEV), torch.zeros(16, device=DEV)
    for bad in (torch.tensor([0.0, 1.0]), [0.5, 1.0], torch.tensor([True, False], device=DEV)):
        with pytest.raises(RuntimeError, match="integers"):
            c.release(bad)
    with pytest.raises(RuntimeError, match="integers"):
        sparse_attn4(q, None, c, sink, None, torch.zeros(1, 1, 4, device=DEV), 1.0)
    for name in ("pool", "table", "refs"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    on = torch.tensor([0, 1], device=DEV)
    c.reserve(on, on, on.to(torch.int32))
    for bad in ([0, 1], torch.tensor([0, 1])):
        with pytest.raises(RuntimeError, match="host memory"):
            c.release(bad)


def test_append_strided_rows_and_far_offsets():
    """Rows cut out of wider ones; and a page whose bytes stand past 2^32 of the pool."""
    from dsv41_amd.kv4 import PagedKV4
    pages = (1 << 32) // (256 * 288) + 40
    pool = torch.zeros(pages, 256, 288, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[[pages - 1, 3]] = 1
    c = PagedKV4(pool, table, refs, dim=512)
    g = _gen(9)
    wide = _rows(g, 10, 1024).to(DEV)
    x = wide[:, 256:768]
    row = torch.tensor([0, 255, 256, 511, 100, 101, 102, 103, 104, 300])
    c.append(x, [0] * 10, row, 1, None, None, 0)
    assert torch.equal(c.read([0] * 10, row).double().cpu(), R.grid(x.double().cpu())[0])
    # and the attention over it
    q = torch.randn(1, 1, 16, 512, generator=g).to(BF)
    from dsv41_amd.kv4 import sparse_attn4
    sink = torch.zeros(16)
    o = sparse_attn4(q.to(DEV), None, c, sink.to(DEV), None, row.to(torch.int32).view(1, 1, -1).to(DEV), 0.05)
    rows = R.grid(x.double().cpu())[0]
    _close(o[0, 0], R.attend(q[0, 0].double(), rows, sink.double(), 0.05), rows.abs().max())


# ------------------------------------------------------------------------------------------------ attention
def _decode(dim, heads, counts, drafts, t, W=128, page=16, seed=0, mask=None, scale=None, qmul=1.0, rd=None):
    from dsv41_amd.kv4 import sattn4
    g = _gen(seed + 31 * t + heads)
    rd = (64 if dim == 512 else 0) if rd is None else rd
    c, rows = _filled(g, counts, dim, page)
    S = len(counts)
    ctx = [max(2 * n + 1, drafts) for n in counts]
    pos = torch.tensor([ctx[s] - drafts + j for s in range(S) for j in range(drafts)])
    seq = torch.tensor([s for s in range(S) for _ in range(drafts)])
    pmax = torch.tensor(ctx)[seq] - 1
    B = len(pos)
    q = (torch.randn(B, 1, heads, dim, generator=g) * qmul).to(BF)
    ring = (torch.randn(S, W, dim, generator=g) * 0.7).to(BF)
    sink = torch.randn(heads, generator=g)
    cos, sin = _angles(max(ctx) + 1, max(rd, 2))
    idx = torch.full((B, 1, t), -1, dtype=torch.int32)
    for b in range(B):
        n = counts[seq[b]]
        k = min(n, t)
        idx[b, 0, :k] = torch.randperm(n, generator=g)[:k].sort().values.to(torch.int32)
    if mask is not None:
        mask(idx, pos, pmax)
    scale = dim ** -0.5 if scale is None else scale
    D = lambda x: x.to(DEV)  # noqa: E731
    o = sattn4(D(q), D(ring), c, D(idx), D(pos), D(sink), D(cos), D(sin), rd, scale, D(seq), D(pmax))
    ref = torch.zeros(B, heads, 512, dtype=torch.float64)
    top = 0.0
    for b in range(B):
        s = int(seq[b])
        keep = idx[b, 0].long()
        keep = keep[(keep >= 0) & (keep < counts[s])]
        k = torch.cat((ring[s][R.ring_slots(int(pos[b]), int(pmax[b]), int(pos[b]), W)].double(), rows[s][keep]))
        top = max(top, k.abs().max().item() if len(k) else 0.0)
        ref[b] = R.rotate(R.attend(q[b, 0].double(), k, sink.double(), scale), cos, sin, int(pos[b]), rd, True) if rd else \
            R.attend(q[b, 0].double(), k, sink.double(), scale)
    assert o.shape == (B, 1, heads, 512)
    _close(o[:, 0], ref, top)
    return o


@pytest.mark.parametrize("dim", [512, 576])
@pytest.mark.parametrize("heads,counts,drafts,t", [
    (64, [300], 1, 512), (64, [1], 1, 1), (64, [0], 1, 7), (16, [65, 0, 700], 1, 64), (20, [129, 40], 2, 65),
    (1, [200], 1, 63), (128, [500, 90], 3, 130), (64, [900] * 5, 6, 257), (8, [60] * 40, 1, 33)])
def test_decode(dim, heads, counts, drafts, t):
    _decode(dim, heads, counts, drafts, t)


@pytest.mark.parametrize("dim,counts,drafts,t", [(576, [2100, 2100], 20, 2048), (512, [1200], 1, 1100), (576, [1000] * 8, 16, 900)])
def test_decode_long_lists(dim, counts, drafts, t):
    """Two workgroups a CU of splits, splits of two tiles, and one split of many."""
    _decode(dim, 64, counts, drafts, t)


@pytest.mark.parametrize("dim", [512, 576])
def test_decode_masks(dim):
    """Entries out of the sequence's pages, holes, a list of nothing, rings that hold nothing yet."""
    def holes(idx, pos, pmax):
        idx[0] = -1
        idx[1, 0, ::3] = -1
        idx[2, 0, 5] = 2 ** 31 - 1
        idx[2, 0, 6] = -2 ** 31
        idx[2, 0, 7] = 100_000
    _decode(dim, 16, [200, 300, 400], 1, 100, mask=holes)

    def nothing(idx, pos, pmax):
        idx[:] = -1
        pmax[:] = -1  # (nothing was written to the ring)
    o = _decode(dim, 64, [100, 90], 1, 70, mask=nothing)
    assert not o.any()


def test_decode_page_sizes_and_windows():
    for page, W in itertools.product((16, 32, 64, 128, 256), (128, 1, 100)):
        _decode(576, 16, [300, 17], 1, 90, W=W, page=page, seed=page + W)


@pytest.mark.parametrize("qmul,scale", [(1.0, 3.0), (1e5, 1e-6), (3e38, 1e-40), (1e-6, 50.0), (0.0, 1.0)])
def test_decode_far_queries(qmul, scale):
    """Logits that differ by hundreds (the running maximum moves), queries past fp16's range and under it.  The ring is
    empty: rows of the cache alone."""
    def no_ring(idx, pos, pmax):
        pmax[:] = -1
    _decode(512, 20, [700, 300], 1, 400, qmul=qmul, scale=scale, mask=no_ring, rd=0)


def test_decode_far_ring():
    """Window rows past fp16's range stay what they are."""
    from dsv41_amd.kv4 import sattn4
    g = _gen(3)
    c, _ = _filled(g, [40], 576, 16)
    ring = torch.zeros(1, 128, 576, dtype=BF)
    ring[0, :, :512] = torch.randn(128, 512, generator=g).to(BF) * 1e30
    q = torch.zeros(1, 1, 16, 576, dtype=BF)
    D = lambda x: x.to(DEV)  # noqa: E731
    one = torch.tensor([300])
    o = sattn4(D(q), D(ring), c, None, D(one), D(torch.full((16,), -1e4)), None, None, 0, 1.0, D(one * 0), D(one - 1))
    ref = ring[0][R.ring_slots(300, 299, 300, 128)].double()[:, :512].mean(0)
    assert ((o[0, 0].double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e30 * 2.0 ** -7).all()


def test_decode_nan_stays_in_its_row():
    """A cache row that holds a NaN reaches the queries that select it, and no other; so does a NaN behind the list."""
    from dsv41_amd.kv4 import sattn4
    g = _gen(4)
    c, _ = _filled(g, [64, 64], 576, 16)
    p = int(c.table[0, 0])
    c.pool[p, 3, 256:288] = 0x7f
    q = torch.randn(3, 1, 20, 576, generator=g).to(BF).to(DEV)
    ring = torch.zeros(2, 128, 576, dtype=BF, device=DEV)
    idx = torch.tensor([[0, 1, 2, 4], [3, 4, 5, 6], [0, 1, 2, 3]], dtype=torch.int32, device=DEV).view(3, 1, 4)
    pos = torch.tensor([200, 200, 200], device=DEV)
    o = sattn4(q, ring, c, idx, pos, torch.zeros(20, device=DEV), None, None, 0, 0.04, torch.tensor([0, 0, 1], device=DEV), pos)
    assert torch.isfinite(o[0]).all() and torch.isnan(o[1]).all() and torch.isfinite(o[2]).all()


def _prefill(dim, heads, b, s, prior, t, w=128, page=16, ratio=4, seed=0, seq=None, strided=False):
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(seed + 7 * s + t)
    n_c = (prior + s) // ratio
    slots = b if seq is None else max(seq) + 1
    c, rows = _filled(g, [n_c] * slots, dim, page)
    hist = min(prior, w - 1)
    q = torch.randn(b, s, heads, dim, generator=g).to(BF)
    kv = (torch.randn(b, hist + s, dim, generator=g) * 0.7).to(BF)
    at = hist + torch.arange(s)[:, None]
    win = (at - w + 1).clamp_min(0) + torch.arange(min(w, hist + s))
    win = torch.where(win <= at, win, -1).to(torch.int32).expand(b, -1, -1).contiguous()
    idx = torch.full((b, s, t), -1, dtype=torch.int32)
    for e in range(b):
        for i in range(s):
            n = (prior + i + 1) // ratio
            k = min(n, t)
            idx[e, i, :k] = torch.randperm(n, generator=g)[:k].sort().values.to(torch.int32)
    sink = torch.randn(heads, generator=g)
    D = lambda x: x.to(DEV)  # noqa: E731
    if strided:
        q = torch.stack((q, q), 2)[:, :, 0]
        both = torch.cat((win, idx), 2).to(DEV)
        wd, xd = both[:, :, :win.shape[2]], both[:, :, win.shape[2]:].long()
        kd = torch.stack((D(kv), D(kv)), 2)[:, :, 1]
    else:
        wd, xd, kd = D(win), D(idx), D(kv)
    sq = None if seq is None else D(torch.tensor(seq))
    o = sparse_attn4(D(q), kd, c, D(sink), wd, xd, dim ** -0.5, seq=sq)
    ref = torch.zeros(b, s, heads, 512, dtype=torch.float64)
    for e in range(b):
        mine = rows[e if seq is None else seq[e]]
        for i in range(s):
            k = torch.cat((kv[e][win[e, i][win[e, i] >= 0].long()].double(), mine[idx[e, i][idx[e, i] >= 0].long()]))
            ref[e, i] = R.attend(q[e, i].double(), k, sink.double(), dim ** -0.5)
    assert o.shape == (b, s, heads, 512)
    _close(o, ref, max(kv.double().abs().max().item(), max(r.abs().max().item() if len(r) else 0 for r in rows)))


@pytest.mark.parametrize("dim", [512, 576])
@pytest.mark.parametrize("heads,b,s,prior,t,w", [
    (64, 1, 1, 0, 16, 128), (64, 1, 37, 0, 16, 128), (20, 2, 21, 130, 40, 128), (8, 1, 70, 500, 130, 128),
    (128, 1, 9, 700, 200, 64), (16, 3, 5, 64, 1, 1), (64, 2, 150, 1001, 65, 128)])
def test_prefill(dim, heads, b, s, prior, t, w):
    _prefill(dim, heads, b, s, prior, t, w)


def test_prefill_many_rows():
    """Enough rows for one split a row and every workgroup shape of many rows."""
    for heads in (16, 32, 48, 64, 80, 128):
        _prefill(576, heads, 1, 530, 400, 100, seed=heads)
    _prefill(512, 64, 1, 530, 400, 200)


@pytest.mark.parametrize("dim,heads,b,s,prior,t,w,page,seq", [
    (576, 33, 1, 530, 400, 256, 100, 16, None),    # one split, half of the second group's heads
    (576, 64, 1, 530, 400, 256, 1, 32, None),
    (512, 80, 1, 530, 400, 250, 37, 64, None),     # two groups of 64 heads, lists that end inside a tile
    (512, 64, 3, 177, 2500, 257, 128, 16, [4, 0, 2]),
    (576, 64, 2, 65, 4300, 1025, 128, 256, [1, 1]),  # two splits; one sequence twice
    (512, 128, 1, 68, 8200, 2000, 64, 128, None)])
def test_prefill_cache_decoded_first(dim, heads, b, s, prior, t, w, page, seq):
    """2^17 listed rows and more, eight times the cache's: its rows are decoded once and attended to as bf16."""
    assert b * s * t >= 1 << 17
    _prefill(dim, heads, b, s, prior, t, w, page, seed=heads, seq=seq, strided=t % 2 == 1)


def _many(g, dim=576, heads=40, s=520, t=260, n=200, page=16):
    """A call whose cache is decoded first: q, the cache with a hole, its rows, lists with rows of the hole and none."""
    c, rows = _filled(g, [n, n], dim, page)
    c.table[1, 3] = -1
    q = torch.randn(1, s, heads, dim, generator=g).to(BF)
    idx = torch.randint(0, n + 30, (1, s, t), generator=g, dtype=torch.int32)
    idx[0, :, ::5] = -1
    idx[0, 7] = -1
    idx[0, 8, :] = 3 * page + 2  # (the hole alone)
    idx[0, 9, 3:] = 2 ** 31 - 1
    held = -(-n // page) * page  # (rows behind the last one of a page are there, as zeros)
    there = lambda i: (i >= 0) & (i < held) & (i // page != 3)  # noqa: E731
    return c, torch.cat((rows[1], torch.zeros(held - n, dim, dtype=torch.float64))), q, idx, there


def test_decoded_first_without_a_window():
    """No window; pages that are not there, indices past the table, rows without a key; a sequence out of range."""
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(21)
    c, rows, q, idx, there = _many(g)
    sink = torch.randn(40, generator=g)
    sink[3], sink[4] = -float("inf"), float("inf")
    args = (q.to(DEV), None, c, sink.to(DEV), None, idx.to(DEV), 0.04)
    o = sparse_attn4(*args, seq=torch.tensor([1], device=DEV))
    ref = torch.zeros(1, q.shape[1], 40, 512, dtype=torch.float64)
    for i in range(q.shape[1]):
        k = idx[0, i][there(idx[0, i])].long()
        ref[0, i] = R.attend(q[0, i].double(), rows[k], sink.double().clamp(-1e300, 1e300), 0.04)
    assert not ref[0, 7].any() and not ref[0, 8].any() and ref[0, 9].any()
    _close(o, ref, rows.abs().max().item())
    for bad in (-1, 2, 1 << 40):
        assert not sparse_attn4(*args, seq=torch.tensor([bad], device=DEV)).any()


def test_decoded_first_nan_stays_in_its_rows():
    """A query of NaN, a cache row of NaN and one of an infinity in the window: the queries that name them and no other."""
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(22)
    c, rows, q, idx, there = _many(g)
    c.table[1, 3] = c.table[0, 3]
    idx[idx == 5] = 6
    idx[0, 11, 4] = 5
    q[0, 12, 39, 3] = float("nan")
    x = torch.full((1, 576), float("nan"), dtype=BF, device=DEV)
    c.append(x, [1], [5], 1, None, None, 0)
    kv = torch.randn(1, 9, 576, generator=g).to(BF)
    kv[0, 8, 575] = float("inf")
    win = torch.randint(-1, 8, (1, q.shape[1], 6), generator=g, dtype=torch.int32)
    win[0, 13, 2] = 8
    o = sparse_attn4(q.to(DEV), kv.to(DEV), c, torch.zeros(40, device=DEV), win.to(DEV), idx.to(DEV), 0.04,
                     seq=torch.tensor([1], device=DEV)).cpu()
    nan = torch.isnan(o[0]).any(-1)
    # (a key column of infinity: a score of -inf is no key, one of +inf leaves inf - inf)
    assert nan[11].all() and nan[12, 39] and not nan[12, :39].any() and torch.equal(nan[13], q[0, 13, :, 575] > 0)
    nan[11:14] = False
    assert not nan.any()


def test_decoded_first_from_a_graph():
    """Captured with the lists and rows that it decodes; replayed on others, against the eager call."""
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(23)
    c, rows, q, idx, there = _many(g)
    q, idx, sink = q.to(DEV), idx.to(DEV), torch.zeros(40, device=DEV)
    seq = torch.tensor([1], device=DEV)
    run = lambda: sparse_attn4(q, None, c, sink, None, idx, 0.04, seq=seq)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g).to(BF))
        idx.copy_(torch.randint(-1, 220, idx.shape, generator=g, dtype=torch.int32))
        seq.fill_(i % 2)
        c.append(_rows(g, 3, 576).to(DEV), [0, 1, 1], [i, i, 40 + i], 1, None, None, 0)
        graph.replay()
        assert torch.equal(out, run()), i


def test_prefill_sequences_and_strides():
    _prefill(576, 16, 2, 11, 90, 30, seq=[3, 1])
    _prefill(512, 64, 2, 11, 90, 30, strided=True)


def test_prefill_lists_of_nothing():
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(8)
    c, rows = _filled(g, [50], 576, 16)
    q = torch.randn(1, 4, 64, 576, generator=g).to(BF).to(DEV)
    sink = torch.zeros(64, device=DEV)
    assert not sparse_attn4(q, None, c, sink, None, None, 0.04).any()
    kv = torch.randn(1, 4, 576, generator=g).to(BF)
    none = torch.full((1, 4, 9), -1, dtype=torch.int32, device=DEV)
    assert not sparse_attn4(q, kv.to(DEV), c, sink, none, none, 0.04).any()
    assert not sparse_attn4(q, kv.to(DEV), c, torch.full((64,), -float("inf"), device=DEV), none, none, 0.04).any()
    # the window alone; indices past its end are none
    win = torch.tensor([[[0, 1, 2, 3, 4, 2 ** 31 - 1]]], dtype=torch.int32).expand(1, 4, 6)
    o = sparse_attn4(q, kv.to(DEV), c, sink, win.to(DEV), None, 0.04)
    ref = torch.stack([R.attend(q[0, i].double().cpu(), kv[0].double(), torch.zeros(64).double(), 0.04) for i in range(4)])
    _close(o[0], ref, kv.double().abs().max())
    assert sparse_attn4(q[:, :0], kv.to(DEV), c, sink, none[:, :0], none[:, :0], 0.04).shape == (1, 0, 64, 512)


def test_same_result_every_time():
    g = _gen(12)
    from dsv41_amd.kv4 import sattn4
    c, _ = _filled(g, [900, 400, 30], 576, 64)
    q = torch.randn(3, 1, 64, 576, generator=g).to(BF).to(DEV)
    ring = torch.randn(3, 128, 576, generator=g).to(BF).to(DEV)
    idx = torch.stack([torch.randperm(900, generator=g)[:600] for _ in range(3)]).to(torch.int32).view(3, 1, -1).to(DEV)
    seq = torch.arange(3, device=DEV)
    pos = torch.tensor([3600, 1700, 122], device=DEV)
    args = (ring, c, idx, pos, torch.zeros(64, device=DEV), None, None, 0, 0.04, seq, pos)
    first = sattn4(q, *args)
    for _ in range(20):
        assert torch.equal(sattn4(q, *args), first)


# ------------------------------------------------------------------------------------------------ pages
def _checked(c, m, data=True):
    assert np.array_equal(c.table.cpu().numpy(), m.table)
    refs = c.refs.cpu().numpy()
    assert np.array_equal(refs, m.refs())
    if data:
        got = c.pool[:, :, 0].cpu().numpy()
        for p in range(m.pages):
            if refs[p]:
                assert list(got[p]) == m.data[p], p


@pytest.mark.parametrize("pages,slots,cols,page,seed", [(40, 6, 9, 16, 0), (40, 6, 9, 16, 1), (300, 30, 20, 32, 2),
                                                        (9000, 40, 300, 16, 3), (20000, 12, 1100, 16, 4)])
def test_pages_against_lists(pages, slots, cols, page, seed):
    """Random calls, each held against lists.  A page's rows carry a mark in their first byte."""
    from dsv41_amd.kv4 import PagedKV4
    rng = random.Random(seed)
    c = PagedKV4(torch.zeros(pages, page, 288, dtype=torch.uint8, device=DEV),
                 torch.full((slots, cols), -1, dtype=torch.int32, device=DEV),
                 torch.zeros(pages, dtype=torch.int32, device=DEV), dim=512)
    m = R.Model(pages, slots, cols, page)
    marks = torch.randint(0, 256, (pages, page), generator=_gen(seed), dtype=torch.uint8)
    c.pool[:, :, 0] = marks.to(DEV)
    for p in range(pages):
        m.data[p] = marks[p].tolist()
    ok = True
    for _ in range(25):
        op = rng.choice(["reserve", "reserve", "reserve", "fork", "release", "compact"])
        if op == "reserve":
            seq = rng.sample(range(slots), rng.randint(1, slots))
            most = cols * page if rng.random() < 0.2 else cols * page // 6
            begin = [rng.randint(0, cols * page) for _ in seq]
            end = [min(cols * page, b + rng.randint(0, most)) for b in begin]
            ok &= m.reserve(seq, begin, end)
            c.reserve(seq, begin, end)
        elif op == "fork":
            both = rng.sample(range(slots), slots)
            k = rng.randint(1, max(1, slots // 2))
            dst, src = both[:k], [rng.choice(both[k:]) for _ in range(k)]
            rows = [rng.randint(0, cols * page) for _ in dst]
            m.fork(src, dst, rows)
            c.fork(src, dst, rows)
        elif op == "release":
            seq = rng.sample(range(slots), rng.randint(1, max(1, slots // 2)))
            rows = [rng.choice([0, rng.randint(0, cols * page)]) for _ in seq]
            m.release(seq, rows)
            c.release(seq, rows)
        else:
            assert int(c.compact()) == m.compact()
        _checked(c, m, data=pages < 1000)
    if ok:
        c.check()
    else:
        with pytest.raises(RuntimeError, match="free pages"):
            c.check()


def test_pages_named_twice_or_out_of_range():
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(30, 6, 100, 512, 16, DEV)
    c.reserve([0, 1], [0, 0], [40, 20])
    c.check()
    for call in (lambda: c.reserve([2, 9], [0, 0], [16, 16]), lambda: c.reserve([3, 3], [0, 0], [16, 32]),
                 lambda: c.reserve([4, -1], [0, 0], [1, 1]), lambda: c.reserve([5], [0], [10_000]),
                 lambda: c.reserve([5], [-1], [4]), lambda: c.release([77]), lambda: c.fork([0], [0]),
                 lambda: c.fork([0, 2], [2, 4]), lambda: c.fork([0, 1], [5, 5]), lambda: c.fork([0], [-2])):
        call()
        with pytest.raises(RuntimeError, match="left out"):
            c.check()
    t = c.table.cpu()
    assert (t[2, 0] >= 0) and (t[3, 0] >= 0) and t[3, 1] < 0 and t[4, 0] == t[2, 0]  # (4 forked from 2, not 2 from 0)
    assert torch.equal(t[5], t[0])
    refs = torch.bincount(t[t >= 0].long(), minlength=30)
    assert torch.equal(refs, c.refs.cpu().long())
    c.release([0, 0, 1], [16, 0, 0])  # (a sequence named twice)
    t = c.table.cpu()
    assert (t[0] < 0).all() and torch.equal(torch.bincount(t[t >= 0].long(), minlength=30), c.refs.cpu().long())


def test_copy_on_write_keeps_the_parent():
    from dsv41_amd.kv4 import PagedKV4
    g, dim = _gen(2), 576
    c = PagedKV4.empty(64, 8, 200, dim, 32, DEV)
    c.reserve([0], [0], [77])
    x = _rows(g, 77, dim).to(DEV)
    c.append(x, [0] * 77, list(range(77)), 1, None, None, 0)
    was = c.read([0] * 77, list(range(77)))
    c.fork([0] * 3, [1, 2, 3], [77, 64, 50])
    c.reserve([1, 2, 3], [77, 64, 50], [80, 70, 60])
    for s, b in ((1, 77), (2, 64), (3, 50)):
        y = _rows(g, 3, dim).to(DEV)
        c.append(y, [s] * 3, [b, b + 1, b + 2], 1, None, None, 0)
        assert torch.equal(c.read([s] * b, list(range(b))), was[:b])
        assert torch.equal(c.read([s] * 3, [b, b + 1, b + 2]).double().cpu(), R.grid(y.double().cpu())[0])
    assert torch.equal(c.read([0] * 77, list(range(77))), was)
    c.release([0, 2])
    c.compact()
    assert torch.equal(c.read([1] * 77, list(range(77))), was) and torch.equal(c.read([3] * 50, list(range(50))), was[:50])
    c.check()


@pytest.mark.parametrize("n,pages", [(1, 3), (50, 64), (1024, 1500), (1025, 1500), (3000, 5000), (4096, 5000),
                                     (4097, 5000), (16385, 17000)])
def test_copy_pages(n, pages):
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(n)
    a, b = (PagedKV4(torch.randint(0, 256, (p, 16, 336), generator=g, dtype=torch.uint8).to(DEV),
                     torch.full((1, 1), -1, dtype=torch.int32, device=DEV), torch.zeros(p, dtype=torch.int32, device=DEV))
            for p in (pages, pages + 7))
    src, dst = torch.randperm(pages, generator=g)[:n], torch.randperm(pages + 7, generator=g)[:n]
    want = b.pool.clone()
    want[dst.to(DEV)] = a.pool[src.to(DEV)]
    b.copy_pages(a, src, dst)
    assert torch.equal(b.pool, want)
    b.check()
    # a page named twice, pages that are none, pages out of range
    src2, dst2 = torch.randint(0, pages, (n,), generator=g), torch.randint(0, pages, (n,), generator=g)
    src2[::7], dst2[3::11] = -1, -1
    src2[5::50] = pages
    dst2[6::50] = pages + 7
    ok = (src2 >= 0) & (src2 < pages) & (dst2 >= 0) & (dst2 < pages + 7)
    for i in range(n):
        if ok[i]:
            want[dst2[i]] = a.pool[src2[i]]
    b.copy_pages(a, src2, dst2)
    assert torch.equal(b.pool, want)


# ------------------------------------------------------------------------------------------------ the whole, as it is used
def _serve(c, g, steps, dim=512, S=3):
    """Prompts, samples forked from one, decode steps that append and attend, one leaves, the pool is compacted."""
    from dsv41_amd.kv4 import sattn4
    ratio, W, H = 2, 128, 20
    cos, sin = (t.to(DEV) for t in _angles(2000))
    n = [90, 33]
    rows = {}
    for s in (0, 1):
        c.reserve([s], [0], [n[s]])
        x = _rows(g, n[s], dim).to(DEV)
        c.append(x, [s] * n[s], list(range(n[s])), ratio, cos, sin, 64)
        y = R.rotate(x.double().cpu(), cos.cpu(), sin.cpu(), torch.arange(n[s]) * ratio, 64).to(BF).double()
        rows[s] = R.grid(y)[0]
    c.fork([0], [2], [70])
    rows[2] = rows[0][:70]
    outs = []
    for step in range(steps):
        live = [s for s in range(S) if s in rows]
        count = [len(rows[s]) for s in live]
        c.reserve(live, count, [k + 1 for k in count])
        x = _rows(g, len(live), dim).to(DEV)
        c.append(x, live, count, ratio, cos, sin, 64)
        for i, s in enumerate(live):
            y = R.rotate(x[i:i + 1].double().cpu(), cos.cpu(), sin.cpu(), torch.tensor([count[i] * ratio]), 64).to(BF).double()
            rows[s] = torch.cat((rows[s], R.grid(y)[0]))
        q = torch.randn(len(live), 1, H, dim, generator=g).to(BF)
        ring = torch.randn(S, W, dim, generator=g).to(BF)
        idx = torch.full((len(live), 1, 60), -1, dtype=torch.int32)
        for i, s in enumerate(live):
            k = min(60, len(rows[s]))
            idx[i, 0, :k] = torch.randperm(len(rows[s]), generator=g)[:k].sort().values.to(torch.int32)
        pos = torch.tensor([2 * len(rows[s]) for s in live])
        seq = torch.tensor(live)
        sink = torch.randn(H, generator=g)
        o = sattn4(q.to(DEV), ring.to(DEV), c, idx.to(DEV), pos.to(DEV), sink.to(DEV), cos, sin, 64, 0.05, seq.to(DEV), pos.to(DEV))
        for i, s in enumerate(live):
            p = int(pos[i])
            k = torch.cat((ring[s][R.ring_slots(p, p, p, W)].double(), rows[s][idx[i, 0][idx[i, 0] >= 0].long()]))
            ref = R.rotate(R.attend(q[i, 0].double(), k, sink.double(), 0.05), cos.cpu(), sin.cpu(), p, 64, True)
            _close(o[i, 0], ref, k.abs().max().item())
        outs.append(o)
        if step == 3:
            c.release([0])
            del rows[0]
            c.compact()
    c.check()
    return outs


def test_together():
    from dsv41_amd.kv4 import PagedKV4
    _serve(PagedKV4.empty(40, 3, 400, 512, 16, DEV), _gen(77), 8)


def test_together_on_another_stream():
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(40, 3, 400, 512, 16, DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _serve(c, _gen(78), 6)
    torch.cuda.current_stream().wait_stream(s)


def test_captured_step():
    """A step -- pages, rows, attention -- captured once and replayed on new contents, with eager work between, against the
    same step run eagerly; two graphs of two caches replayed in turn."""
    from dsv41_amd.kv4 import PagedKV4, sattn4
    g, dim, H, B = _gen(55), 576, 64, 4
    seq = torch.arange(B, device=DEV)
    made = []
    for k in range(2):
        a, b = (PagedKV4.empty(60, 5, 300, dim, 16, DEV) for _ in range(2))
        st = dict(x=torch.zeros(B, dim, dtype=BF, device=DEV), row=torch.zeros(B, dtype=torch.int64, device=DEV),
                  end=torch.ones(B, dtype=torch.int64, device=DEV), q=torch.zeros(B, 1, H, dim, dtype=BF, device=DEV),
                  ring=torch.randn(B, 128, dim, generator=g).to(BF).to(DEV), pos=torch.zeros(B, dtype=torch.int64, device=DEV),
                  idx=torch.full((B, 1, 150), -1, dtype=torch.int32, device=DEV), sink=torch.randn(H, generator=g).to(DEV))

        def step(c, st=st):
            c.reserve(seq, st["row"], st["end"])
            c.append(st["x"], seq, st["row"], 4, None, None, 0)
            o = sattn4(st["q"], st["ring"], c, st["idx"], st["pos"], st["sink"], None, None, 0, 0.05, seq, st["pos"])
            return o, c.read(seq, st["row"])
        # (captured on a cache's state before any row: the capture itself runs nothing)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(PagedKV4.empty(60, 5, 300, dim, 16, DEV))
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(a)
        made.append((a, b, st, step, graph, out))
    for i in range(6):
        for a, b, st, step, graph, out in made:
            st["x"].copy_(_rows(g, B, dim).to(DEV))
            st["row"].fill_(i * 7)
            st["end"].fill_(i * 7 + 1)
            st["q"].copy_(torch.randn(B, 1, H, dim, generator=g).to(BF).to(DEV))
            st["pos"].fill_(i * 28 + 3)
            st["idx"][:, 0, :i + 1] = torch.arange(i + 1, device=DEV) * 7
        for a, b, st, step, graph, out in made:
            graph.replay()
        torch.cuda.synchronize()
        for a, b, st, step, graph, out in made:
            want = step(b)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
            assert torch.equal(a.table, b.table) and torch.equal(a.refs, b.refs) and torch.equal(a.pool, b.pool)
    for a, b, *_ in made:
        a.check()


# ------------------------------------------------------------------------------------------------ in the layers
def _layer_weights(g, dim, q_rank, H, D, HI):
    n = lambda *s: torch.randn(*s, generator=g) * s[-1] ** -0.5  # noqa: E731
    w = dict(wq_a=n(q_rank, dim), q_norm_w=1 + 0.1 * n(q_rank), wq_b=n(H * D, q_rank), wkv=n(D, dim), kv_norm_w=1 + 0.1 * n(D),
             c_norm_w=1 + 0.1 * n(D), i_wq_b=n(HI * 128, q_rank), i_weights_proj=n(HI, dim), i_wk=n(128, D),
             i_k_norm_w=1 + 0.1 * n(128))
    w = {k: v.to(BF).to(DEV) for k, v in w.items()}
    w.update(c_wkv=n(D, dim).to(DEV), c_wgate=n(D, dim).to(DEV), attn_sink=torch.randn(H, generator=g).to(DEV))
    return w


def _alike(a, b, most):
    """Two outputs that are each off by 2^-8 (|o| + V), V the largest value (see _close), then rotated -- sqrt 2 of it at
    most -- and rounded again: 7 2^-8 V apart; as a whole by twice 2^-8 of the norm and two roundings."""
    a, b = a.double(), b.double()
    assert torch.isfinite(a).all() and (a - b).abs().max() <= 7 * 2.0 ** -8 * most
    assert (a - b).norm() <= 3 * 2.0 ** -8 * b.norm()


@pytest.mark.parametrize("b", [1, 2])
def test_attention_layer_over_a_4_bit_cache(b):
    """SparseAttention with its compressed rows in a PagedKV4 beside one with the bf16 table, over a prompt, a
    continuation that selects, steps that close a group and steps that do not, and a second prompt in the same slots."""
    from dsv41_amd.attention import SparseAttention
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(40 + b)
    dim, q_rank, H, D, HI, ratio, cap = 256, 128, 20, 512, 16, 2, 400
    w = _layer_weights(g, dim, q_rank, H, D, HI)
    cos, sin = (t.to(DEV) for t in _angles(2 * cap))
    kw = dict(n_heads=H, head_dim=D, rope_head_dim=64, window=32, ratio=ratio, index_n_heads=HI, index_topk_k=100, cos=cos,
              sin=sin, slots=b, cap=cap)
    c = PagedKV4.empty(b * -(-cap // 32), b, cap, D, 32, DEV)
    one, two = SparseAttention(w, **kw), SparseAttention(w, kv4=c, **kw)
    x = torch.randn(b, 700, dim, generator=g).to(BF).to(DEV)
    for lo, hi in ((0, 1), (1, 2), (0, 333), (333, 601), (601, 602), (602, 603), (603, 604), (0, 90)):
        o, p = one.attend(x[:, lo:hi], lo), two.attend(x[:, lo:hi], lo)
        n = hi // ratio
        rows = torch.arange(n, device=DEV).repeat(b)
        got = c.read(torch.arange(b, device=DEV).repeat_interleave(n), rows).view(b, n, D)
        assert (got != one.ckv[:, :n]).any(-1).sum().item() <= 2 * b  # (rotated in fp32 there, in 64 bits here)
        assert torch.equal(one.ring, two.ring)
        _alike(p, o, max(one.ckv.abs().max().item(), one.ring.abs().max().item(), 1.0))
    c.check()
    with pytest.raises(ValueError, match="without compressed rows"):
        SparseAttention(w, kv4=c, **dict(kw, ratio=0))
    with pytest.raises(RuntimeError, match="capacity"):
        two.attend(x[:, :1], 2 * cap + 1)
    for bad in (PagedKV4.empty(9, b, cap, 576, 32, DEV), PagedKV4.empty(9, b, cap - 40, D, 32, DEV)):
        with pytest.raises(ValueError, match="SparseAttention"):
            SparseAttention(w, kv4=bad, **kw)


def test_decode_layer_over_a_4_bit_cache():
    """DecodeLayer with a PagedKV4 in the place of the bf16 table: appends, selection and attention of steps that close a
    group and steps that do not, by both ways of the appends; then the step from a graph."""
    from dsv41_amd.decode import DecodeLayer
    from dsv41_amd.kv4 import PagedKV4
    from dsv41_amd.workloads import DecodeConfig, make_decode_inputs
    cfg = DecodeConfig("T", [8300, 900, 40], topk=512, spare=20)
    (l0,), st = make_decode_inputs(cfg, DEV, seed=9)
    B, cap = 3, l0["ckv"].shape[1]
    cos, sin = (t.to(DEV) for t in _angles(8400))
    c = PagedKV4.empty(B * -(-cap // 64), B, cap, 576, 64, DEV)
    rows = torch.arange(cap, device=DEV).repeat(B)
    seqs = torch.arange(B, device=DEV).repeat_interleave(cap)
    c.reserve([0, 1, 2], [0, 0, 0], [cap] * 3)
    c.append(l0["ckv"], seqs, rows, 1, None, None, 0)
    l0["ckv"] = c.read(seqs, rows).view(B, cap, 576)
    mk = lambda ckv: DecodeLayer(l0["ring"].clone(), ckv, l0["k8"].clone(), l0["ks"].clone(), st["sink"], cos, sin,  # noqa: E731
                                 cfg.ratio, cfg.topk)
    one, two = mk(l0["ckv"].clone()), mk(c)
    g = _gen(10)
    kv_raw, latent, k_raw, pos = st["kv_raw"].clone(), st["latent"].clone(), st["k_raw"].clone(), st["pos"].clone()

    def step(lay, fused):
        a = (kv_raw, st["kv_norm"], latent, k_raw, st["k_norm"], pos, st["seq"], st["q_idx"], st["w_idx"])
        if fused:
            idx = lay.appends_select(*a)
        else:
            lay.appends(*a)
            idx = lay.select(st["q_idx"], st["w_idx"], pos, st["seq"])
        return idx.clone(), lay.attend(st["q"], idx, pos, st["seq"], pos)

    def same(a, b, i):
        assert torch.equal(a[0], b[0]), i
        top = max(l0["ckv"].abs().max().item(), one.ring.abs().max().item(), one.ckv.abs().max().item())
        _alike(b[1], a[1], top)
        cl = ((pos + 1) // cfg.ratio - 1).tolist()
        got = c.read([0, 1, 2], cl)
        want = torch.stack([one.ckv[s, r] for s, r in enumerate(cl)])
        assert (got != want).sum().item() <= 2, i

    def fresh(i):
        kv_raw.copy_(torch.randn(kv_raw.shape, generator=g))
        latent.copy_(torch.randn(latent.shape, generator=g))
        k_raw.copy_(torch.randn(k_raw.shape, generator=g))
        pos.add_(1 if i else 0)

    for i in range(6):
        fresh(i)
        same(step(one, i % 2 == 0), step(two, i % 2 == 0), i)
        one.check(), two.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(two, True)
    for i in range(1, 6):
        fresh(i)
        graph.replay()
        same(step(one, True), out, i)
    two.check()
    c.release([1])
    two.appends(kv_raw, st["kv_norm"], latent, k_raw, st["k_norm"], torch.full_like(pos, 903), st["seq"])
    with pytest.raises(RuntimeError, match="dropped"):
        two.check()
    with pytest.raises(ValueError, match="DecodeLayer"):
        DecodeLayer(l0["ring"], PagedKV4.empty(1, 1, 1, 512, 64, DEV), l0["k8"], l0["ks"], st["sink"], cos, sin, 4, 512)
