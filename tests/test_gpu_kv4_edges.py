"""The paged 4-bit cache at its edges: host memory that changes after a call, queries far below fp16's range, long flat
lists, counts that disagree with the table, unusual views, positions limited by plim, layers whose sequences are forked."""
import pytest
import torch

import _kv4_ref as R
from test_gpu_kv4 import BF, DEV, _alike, _angles, _close, _decode, _filled, _gen, _layer_weights, _rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ index arguments
@pytest.mark.parametrize("pinned", [True, False])
@pytest.mark.parametrize("n", [3, 1 << 20])
def test_host_indices_may_change_after_the_call(pinned, n):
    """A caller that keeps one host buffer fills it for its next step while the GPU still works on earlier ones."""
    from dsv41_amd._lib import as_i64
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(2, 1, 32, 512, 16, DEV)
    busy = torch.randn(4096, 4096, device=DEV)
    for take in (lambda t: c._i64("x", t, n), lambda t: as_i64(t, c.device)):
        t = torch.empty(n, dtype=torch.int64, pin_memory=pinned).fill_(5)
        torch.cuda.synchronize()
        for _ in range(40):
            busy @ busy
        got = take(t)
        t.fill_(9)
        assert bool((got == 5).all())


def test_rows_go_where_a_pinned_index_said():
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(4, 1, 64, 512, 16, DEV)
    c.reserve([0], [0], [64])
    x = torch.full((2, 512), 6.0, dtype=BF, device=DEV)
    seq = torch.zeros(2, dtype=torch.int64, device=DEV)
    row = torch.tensor([3, 20]).pin_memory()
    busy = torch.randn(4096, 4096, device=DEV)
    for _ in range(40):
        busy @ busy
    c.append(x, seq, row, 1, None, None, 0)
    row.copy_(torch.tensor([40, 41]))
    assert c.read([0, 0, 0, 0], [3, 20, 40, 41]).eq(6).all(1).tolist() == [True, True, False, False]


def test_pinned_indices_of_queued_calls_stay_apart():
    """Many calls queued behind a busy stream, from one pinned buffer: asynchronous, and each has its own entries."""
    from dsv41_amd.kv4 import PagedKV4
    c = PagedKV4.empty(2, 1, 32, 512, 16, DEV)
    busy, t = torch.randn(4096, 4096, device=DEV), torch.empty(1 << 16, dtype=torch.int64).pin_memory()
    c._i64("x", t, len(t))
    torch.cuda.synchronize()
    for _ in range(300):
        busy @ busy
    done = torch.cuda.Event()
    done.record()
    got = [c._i64("x", t.fill_(k), len(t)) for k in range(8)]
    assert not done.query()  # (none of them waited)
    assert [(int(g.min()), int(g.max())) for g in got] == [(k, k) for k in range(8)]


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.int8, torch.uint8])
def test_attention_takes_any_integer_list(dtype):
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(31)
    c, _ = _filled(g, [100], 576, 16)
    q = torch.randn(1, 2, 16, 576, generator=g).to(BF).to(DEV)
    kv = torch.randn(1, 9, 576, generator=g).to(BF).to(DEV)
    sink = torch.zeros(16, device=DEV)
    idx, win = torch.randint(0, 100, (1, 2, 40), generator=g), torch.randint(0, 9, (1, 2, 5), generator=g)
    if dtype != torch.uint8:
        idx[0, 1, ::3], win[0, 0, 1] = -1, -1
    run = lambda t: sparse_attn4(q, kv, c, sink, win.to(t).to(DEV), idx.to(t).to(DEV), 0.04)  # noqa: E731
    assert torch.equal(run(dtype), run(torch.int32))


# ------------------------------------------------------------------------------------------------ numbers
@pytest.mark.parametrize("qmul,scale", [(1e-6, 5e4), (1e-9, 3e8), (1e-36, 1e36), (2.0 ** -130, 2.0 ** 127)])
def test_decode_queries_below_fp16(qmul, scale):
    """Queries below fp16's smallest numbers under a scale that makes their logits ordinary ones; the ring is empty."""
    def no_ring(idx, pos, pmax):
        pmax[:] = -1
    _decode(512, 20, [700, 300], 1, 400, qmul=qmul, scale=scale * 0.05, mask=no_ring, rd=0)
    _decode(576, 16, [200], 3, 90, qmul=qmul, scale=scale * 0.05, mask=no_ring, rd=0)


@pytest.mark.parametrize("window", [False, True])
def test_long_list_behind_a_peak(window):
    """One key (of the cache, or of the window) of weight 1, then 2^18 of 2^-25.5 each, 0.55 % of the weight together, over
    one split.  Scores come from column 512, which is no value.  The output is off by its rounding (2^-8 of it), the peak's
    probability's (2^-8 of its value 1.5) and each small one's: 2^-25 where the peak has 2^7 or more, so n 2^-32."""
    from dsv41_amd.kv4 import PagedKV4, sparse_attn4
    n, s = 1 << 18, 520
    rows = torch.zeros(2, 576)
    rows[0, :512], rows[0, 512] = 1.5, 6.0  # (the grid's: 6 times a power of two)
    rows[1, :512] = 6.0
    c = PagedKV4.empty(1, 1, 16, 576, 16, DEV)
    c.reserve([0], [0], [2])
    c.append(rows.to(BF).to(DEV), [0, 0], [0, 1], 1, None, None, 0)
    q = torch.zeros(1, s, 16, 576, dtype=BF, device=DEV)
    q[..., 512] = 1.0
    scale = 25.5 * torch.log(torch.tensor(2.0, dtype=torch.float64)).item() / 6
    idx = torch.ones(1, s, n + 64, dtype=torch.int32, device=DEV)
    idx[:, :, :64] = -1
    kv = win = None
    if window:
        kv, win = rows[:1].to(BF).to(DEV).view(1, 1, 576), torch.zeros(1, s, 1, dtype=torch.int32, device=DEV)
    else:
        idx[:, :, 0] = 0
    o = sparse_attn4(q, kv, c, torch.full((16,), -1e30, device=DEV), win, idx, scale)
    w = n * 2.0 ** -25.5
    want = (1.5 + 6 * w) / (1 + w)
    bound = 2.0 ** -8 * want + 2.0 ** -8 * 1.5 + 6 * n * 2.0 ** -32
    assert (o.double() - want).abs().max().item() <= bound
    assert bound < 0.5 * 6 * w  # (what it leaves out would show)


@pytest.mark.parametrize("H,t", [(1, 63), (3, 200), (16, 63)])
def test_partial_results_stand_aligned(H, t):
    """The splits' partial results: rows of 512 at the workspace's start, 16-byte aligned, whatever the number of rows, heads
    and splits, then their references (in powers of two) and sums; joined here they are the output."""
    from dsv41_amd._lib import lib
    g = _gen(t + H)
    c, _ = _filled(g, [300], 576, 16)
    D = lambda x: x.to(DEV)  # noqa: E731
    q, ring, sink = (D(torch.randn(*s, generator=g)) for s in ((1, H, 576), (1, 128, 576), (H,)))
    q, ring = q.to(BF), ring.to(BF)
    idx = D(torch.randperm(300, generator=g)[:t].to(torch.int32))
    pos, seq = D(torch.tensor([700])), D(torch.tensor([0]))
    size = lib().dsv41_kv4_attn_workspace_bytes(c._at, 1, H, 128, t, 0)
    n = 2 + -(-t // 64)
    assert size == 4 * H * n * 514
    ws, out = torch.zeros(size // 4, device=DEV), torch.zeros(H, 512, dtype=BF, device=DEV)
    rc = lib().dsv41_sattn4(c._at, q.data_ptr(), ring.data_ptr(), 128 * 576, 1, 128, idx.data_ptr(), t, pos.data_ptr(),
                            seq.data_ptr(), pos.data_ptr(), None, sink.data_ptr(), None, None, 0, 0, 0.04, out.data_ptr(), 1, H,
                            ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    o, ml = ws[:H * n * 512].view(H, n, 512).double(), ws[H * n * 512:].view(H, n, 2).double()
    top = ml[..., 0].amax(1)
    w = torch.exp2(ml[..., 0] - top[:, None])
    den = (w * ml[..., 1]).sum(1) + torch.exp2(sink.double() / torch.log(torch.tensor(2.0, dtype=torch.float64)) - top)
    want = (w[..., None] * o).sum(1) / den[:, None]
    # (one rounding to bf16; the powers of two and the sums are off by 2^-20 of their terms)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * ring.double().abs().max()).all()


# ------------------------------------------------------------------------------------------------ pages
def test_compact_of_a_page_without_a_count():
    """A table's entry whose page has no count names no page of another sequence afterwards, whatever the workspace held,
    and is noted."""
    from dsv41_amd._lib import lib
    from dsv41_amd.kv4 import PagedKV4
    pool = torch.randint(0, 256, (9, 16, 288), generator=_gen(1), dtype=torch.uint8).to(DEV)
    table = torch.tensor([[6, 5, -1], [7, -1, 8]], dtype=torch.int32, device=DEV)
    refs = torch.tensor([0, 0, 0, 0, 0, 1, 1, 0, 1], dtype=torch.int32, device=DEV)  # (page 7 is named, but not counted)
    c = PagedKV4(pool.clone(), table.clone(), refs.clone(), dim=512)
    size = lib().dsv41_kv4_compact_workspace_bytes(c._at)
    ws = torch.ones(size // 4, dtype=torch.int32, device=DEV)
    live = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert lib().dsv41_kv4_compact(c._at, live.data_ptr(), ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    assert live.item() == 3 and c.table.tolist() == [[1, 0, -1], [-1, -1, 2]] and c.refs.tolist() == [1] * 3 + [0] * 6
    assert torch.equal(c.pool[:3], pool[[5, 6, 8]])
    with pytest.raises(RuntimeError, match="left out"):
        c.check()


def test_reserve_keeps_the_rows_before_begin_alone():
    """A shared page that is replaced keeps its rows before begin for the sequence; those from begin on are what the new
    page held, until they are appended.  The other sequence's rows stay."""
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(6)
    c = PagedKV4.empty(8, 2, 64, 512, 32, DEV)
    c.reserve([0], [0], [50])
    x = _rows(g, 50, 512).to(DEV)
    c.append(x, [0] * 50, list(range(50)), 1, None, None, 0)
    was = c.read([0] * 50, list(range(50)))
    c.fork([0], [1])
    c.reserve([1], [10], [12])
    y = _rows(g, 2, 512).to(DEV)
    c.append(y, [1, 1], [10, 11], 1, None, None, 0)
    got = c.read([1] * 50, list(range(50)))
    assert torch.equal(got[:10], was[:10]) and torch.equal(got[32:], was[32:])  # (the second page is still shared)
    assert torch.equal(got[10:12].double().cpu(), R.grid(y.double().cpu())[0]) and not got[12:32].any()
    assert torch.equal(c.read([0] * 50, list(range(50))), was)
    c.check()


# ------------------------------------------------------------------------------------------------ views
def test_windows_of_one_batch_row_and_of_none():
    """Window rows of one batch row (or ring) cut out of a wider buffer, whose batch stride is then any number; and a window
    without rows beside a list."""
    from dsv41_amd.kv4 import sattn4, sparse_attn4
    g = _gen(13)
    c, _ = _filled(g, [60], 576, 16)
    q = torch.randn(1, 3, 16, 576, generator=g).to(BF).to(DEV)
    sink = torch.zeros(16, device=DEV)
    wide = torch.randn(128 * 576 + 4, generator=g).to(BF).to(DEV)
    odd = wide.as_strided((1, 128, 576), (128 * 576 + 4, 576, 1))
    assert odd.stride(0) % 8 and odd.is_contiguous()
    idx = torch.randint(0, 60, (1, 3, 20), generator=g, dtype=torch.int32).to(DEV)
    win = torch.randint(0, 128, (1, 3, 9), generator=g, dtype=torch.int32).to(DEV)
    assert torch.equal(sparse_attn4(q, odd, c, sink, win, idx, 0.04), sparse_attn4(q, odd.clone(), c, sink, win, idx, 0.04))
    one = torch.tensor([500], device=DEV)
    step = lambda r: sattn4(q[:, :1], r, c, idx[:, :1], one, sink, None, None, 0, 0.04, one * 0, one)  # noqa: E731
    assert torch.equal(step(odd), step(odd.clone()))
    none = torch.zeros(1, 0, 576, dtype=BF, device=DEV)
    want = sparse_attn4(q, None, c, sink, None, idx, 0.04)
    assert torch.equal(sparse_attn4(q, none, c, sink, win, idx, 0.04), want) and want.any()
    assert not sparse_attn4(q, none, c, sink, win, None, 0.04).any()


# ------------------------------------------------------------------------------------------------ attention, row by row
def _each(o, q, keys, sink, scale, splits=1):
    """Every (row, head) by its own norm.  Probabilities in bf16 (2^-8 of each), partial results in bf16 where a row is split,
    one rounding: 2^-8 |o| + splits 2^-8 sum p |v|; fp32 logits are off by 2^-20 of the largest, which adds that to every p.
    keys[i]: the rows that query i sees, fp64."""
    bad = 0
    for i in range(len(q)):
        x = torch.cat((q[i].double() @ keys[i].t() * scale, sink.double()[:, None]), 1)
        p, v = x.softmax(1)[:, :-1], keys[i][:, :512]
        ref = p @ v
        rel = splits * 2.0 ** -8 + 2.0 ** -19 * x.abs().max()
        bound = 2.0 ** -8 * ref.norm(dim=1) + rel * (p * v.norm(dim=1)).sum(1)
        bad += int(((o[i].double().cpu() - ref).norm(dim=1) > bound).sum())
    assert bad == 0


@pytest.mark.parametrize("dim,heads,s,prior,t", [(576, 40, 530, 400, 256), (512, 16, 90, 900, 200), (576, 20, 40, 900, 100)])
def test_prompt_row_by_row(dim, heads, s, prior, t):
    """Sharp softmaxes, so that a few keys are most of each (row, head), at other places of the list for each: a wrong one
    among them is more than the 2 % that its norm may be off by."""
    from dsv41_amd.kv4 import sparse_attn4
    g = _gen(s + heads)
    n = (prior + s) // 4
    c, (rows,) = _filled(g, [n], dim, 16)
    q = torch.randn(1, s, heads, dim, generator=g).to(BF)
    kv = (torch.randn(1, s, dim, generator=g) * 0.7).to(BF)
    win = (torch.arange(s)[:, None] - torch.arange(100)).to(torch.int32)[None]
    idx = torch.full((1, s, t), -1, dtype=torch.int32)
    for i in range(s):
        k = min(n, t)
        idx[0, i, :k] = torch.randperm(n, generator=g)[:k].to(torch.int32)
    sink = torch.randn(heads, generator=g)
    o = sparse_attn4(q.to(DEV), kv.to(DEV), c, sink.to(DEV), win.clamp_min(-1).to(DEV), idx.to(DEV), 0.5)
    keys = [torch.cat((kv[0].double()[win[0, i][win[0, i] >= 0].long()], rows[idx[0, i][idx[0, i] >= 0].long()])) for i in range(s)]
    _each(o[0], q[0], keys, sink, 0.5, splits=2)


@pytest.mark.parametrize("dim", [512, 576])
def test_drafts_see_up_to_plim(dim):
    """Rows of one sequence whose ring already holds later positions, each limited by its own plim: all of them, some, none."""
    from dsv41_amd.kv4 import sattn4
    g = _gen(dim + 5)
    W, H, rd = 128, 20, 64 if dim == 512 else 0
    c, rows = _filled(g, [260, 40], dim, 16)
    pos = torch.tensor([600, 601, 602, 603, 90, 91, 127, 604])
    seq = torch.tensor([0, 0, 0, 0, 1, 1, 1, 0])
    pmax = torch.tensor([603, 603, 603, 603, 127, 127, 127, 603])
    plim = torch.tensor([600, 601, 550, 603, 90, 40, -1, 500])
    B = len(pos)
    q = torch.randn(B, 1, H, dim, generator=g).to(BF)
    ring = (torch.randn(2, W, dim, generator=g) * 0.7).to(BF)
    idx = torch.stack([torch.randperm(40, generator=g)[:30] for _ in range(B)]).to(torch.int32).view(B, 1, 30)
    sink = torch.randn(H, generator=g)
    cos, sin = _angles(700)
    D = lambda x: x.to(DEV)  # noqa: E731
    call = lambda lim: sattn4(D(q), D(ring), c, D(idx), D(pos), D(sink), D(cos), D(sin), rd, 0.5, D(seq), D(pmax), lim)  # noqa: E731
    o = call(D(plim))
    keys, turned = [], o[:, 0].double().cpu()
    for b in range(B):
        e = int(seq[b])
        seen = R.ring_slots(int(pos[b]), int(pmax[b]), int(plim[b]), W)
        keys.append(torch.cat((ring[e][seen].double(), rows[e][idx[b, 0].long()])))
        if rd:  # (turned back: a rotation keeps the norm that is looked at)
            turned[b] = R.rotate(turned[b], cos, sin, int(pos[b]), rd)
    assert len({len(k) for k in keys}) > 4
    _each(turned, q[:, 0], keys, sink, 0.5)
    assert torch.equal(call(None), call(D(pos))) and torch.equal(call(D(plim.to(torch.int32))), o)


def test_positions_outside_the_rope_tables():
    """The rotated columns of a row whose position has no angle are NaN; its others and the other rows are what they are."""
    from dsv41_amd.kv4 import sattn4
    g = _gen(17)
    c, _ = _filled(g, [80], 512, 16)
    q = torch.randn(4, 1, 16, 512, generator=g).to(BF).to(DEV)
    ring = torch.randn(1, 128, 512, generator=g).to(BF).to(DEV)
    idx = torch.randint(0, 80, (4, 1, 70), generator=g, dtype=torch.int32).to(DEV)
    pos = torch.tensor([199, 200, 198, 1 << 30], device=DEV)
    zero, sink = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(16, device=DEV)
    run = lambda n: sattn4(q, ring, c, idx, pos, sink, *(t.to(DEV) for t in _angles(n)), 64, 0.04, zero, zero + 199)  # noqa: E731
    o, plain = run(200)[:, 0], run(201)[:, 0]
    assert torch.equal(torch.isnan(o).any(1).any(1).cpu(), torch.tensor([False, True, False, True]))
    assert torch.isnan(o[[1, 3], :, 448:]).all() and torch.equal(o[..., :448], plain[..., :448])
    assert torch.equal(o[[0, 2]], plain[[0, 2]]) and torch.isfinite(plain[1]).all()


# ------------------------------------------------------------------------------------------------ in the layer
def test_attention_layer_forks_a_sequence():
    """A sequence of the layer forked as its documentation says -- the pages by fork, the other tables' rows copied -- and
    both go on apart, beside a layer over a bf16 table whose rows were all copied."""
    from dsv41_amd.attention import SparseAttention
    from dsv41_amd.kv4 import PagedKV4
    g = _gen(91)
    dim, q_rank, H, D, HI, cap = 256, 128, 20, 512, 16, 300
    w = _layer_weights(g, dim, q_rank, H, D, HI)
    cos, sin = (t.to(DEV) for t in _angles(2 * cap))
    kw = dict(n_heads=H, head_dim=D, rope_head_dim=64, window=32, ratio=2, index_n_heads=HI, index_topk_k=60, cos=cos, sin=sin,
              slots=2, cap=cap)
    c = PagedKV4.empty(24, 2, cap, D, 32, DEV)
    one, two = SparseAttention(w, **kw), SparseAttention(w, kv4=c, **kw)
    x = torch.randn(2, 420, dim, generator=g).to(BF).to(DEV)
    most = lambda: max(one.ckv.abs().max().item(), one.ring.abs().max().item(), 1.0)  # noqa: E731
    _alike(two.attend(x[:, :301], 0), one.attend(x[:, :301], 0), most())
    for lay in (one, two):
        for t in (lay.ring, lay.index_k, lay.k8, lay.ks, lay.ring_kv, lay.ring_score):
            t[1] = t[0]
    one.ckv[1] = one.ckv[0]
    c.fork([0], [1])
    for lo, hi in ((301, 302), (302, 303), (303, 350), (350, 420)):
        _alike(two.attend(x[:, lo:hi], lo), one.attend(x[:, lo:hi], lo), most())
    c.check()
    assert (c.refs > 1).any()  # (whole pages of the prefix are still shared)
    n = 420 // 2
    got = c.read(torch.arange(2, device=DEV).repeat_interleave(n), torch.arange(n, device=DEV).repeat(2)).view(2, n, D)
    assert (got != one.ckv[:, :n]).any(-1).sum().item() <= 4  # (rotated in fp32 there, in 64 bits here)
