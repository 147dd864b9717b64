"""The paged 4-bit cache on the CPU: what its calls refuse, workspace sizes, and the tests' own 64-bit forms."""
import numpy as np
import pytest
import torch

import _kv4_ref as R
from dsv41_amd import _lib, kv4

BF = torch.bfloat16


def _tensors(pages=4, page=16, slots=2, cols=3, dim=512):
    return (torch.zeros(pages, page, R.ROW_BYTES[dim], dtype=torch.uint8), torch.full((slots, cols), -1, dtype=torch.int32),
            torch.zeros(pages, dtype=torch.int32))


def test_cache_refuses():
    pool, table, refs = _tensors()
    with pytest.raises(RuntimeError, match="GPU"):
        kv4.PagedKV4(pool, table, refs, dim=512)
    with pytest.raises(RuntimeError, match="GPU"):
        kv4.PagedKV4.empty(4, 2, 30, 512, 16, "cpu")
    bad = [dict(dim=576), dict(dim=500), dict(pool=pool.int()), dict(pool=pool[:, :15]), dict(pool=pool[:, :, :280]),
           dict(table=table.long()), dict(table=table[0]), dict(refs=refs.long()), dict(refs=refs[:3]),
           dict(table=table[:, :0]), dict(table=table.t()), dict(pool=torch.zeros(4, 32, 288, dtype=torch.uint8)[:, ::2])]
    for b in bad:
        with pytest.raises(ValueError):
            kv4.PagedKV4(**{**dict(pool=pool, table=table, refs=refs, dim=512), **b})
    for b in [(0, 2, 30, 512, 16), (4, 0, 30, 512, 16), (4, 2, 0, 512, 16), (4, 2, 30, 64, 16), (4, 2, 30, 512, 48)]:
        with pytest.raises(ValueError):
            kv4.PagedKV4.empty(*b)


def _cache(dim=576):
    """A cache's handle without a GPU behind it, to reach the checks of arguments (no call below gets past them)."""
    c = kv4.PagedKV4.__new__(kv4.PagedKV4)
    c.pool, c.table, c.refs = _tensors(dim=dim)
    c.dim, c.pages, c.page, c.slots, c.cols, c.device = dim, 4, 16, 2, 3, torch.device("cpu")
    return c


def test_calls_refuse():
    c = _cache()
    x, cs = torch.zeros(2, 576, dtype=BF), torch.zeros(8, 32)
    i = torch.zeros(2, dtype=torch.int64)
    for bad in [(x.float(), i, i, 4, cs, cs, 64), (x[:, :512], i, i, 4, cs, cs, 64), (x, i, i, 0, cs, cs, 64),
                (x, i, i, 4, cs, cs, 63), (x, i, i, 4, cs, cs, 578), (x, i, i, 4, cs, cs, 64)]:
        with pytest.raises(RuntimeError):
            c.append(*bad)
    with pytest.raises(RuntimeError, match="beside"):
        c._i64("x", 2, i, torch.zeros(3))
    with pytest.raises(RuntimeError, match="at most"):
        c.reserve(torch.zeros(4097), torch.zeros(4097), torch.zeros(4097))
    with pytest.raises(RuntimeError, match="pages of"):
        c.copy_pages(_cache(512), i, i)
    q, ring = torch.zeros(2, 1, 4, 576, dtype=BF), torch.zeros(2, 128, 576, dtype=BF)
    sink = torch.zeros(4)
    for f in (lambda: kv4.sattn4(q, ring, c, None, i, sink, None, None, 0, 1.0, i, i),
              lambda: kv4.sattn4(q.expand(2, 2, 4, 576), ring, c, None, i, sink, None, None, 0, 1.0, i, i),
              lambda: kv4.sattn4(q, ring, c, None, i, sink, None, None, 0, 1.0, i, i, d_v=576),
              lambda: kv4.sparse_attn4(q, None, c, sink, None, None, 1.0),
              lambda: kv4.sparse_attn4(q, None, c, sink, None, None, 1.0, d_v=128)):
        with pytest.raises(RuntimeError):
            f()
    with pytest.raises(TypeError):
        kv4.sparse_attn4(q, None, c.pool, sink, None, None, 1.0)


def test_indices_and_windows_refuse():
    with pytest.raises(RuntimeError, match="indices"):
        kv4._indices("x", torch.zeros(2, 3, 4), (2, 2), -1)
    assert kv4._indices("x", torch.zeros(2, 2, 0, dtype=torch.int32), (2, 2), -1) == (None, 0)
    got, t = kv4._indices("x", torch.tensor([[[1 << 40, -(1 << 40), 5]]]), (1, 1), -1)
    assert t == 3 and got.tolist() == [[[2 ** 31 - 1, -1, 5]]]
    for kv in (torch.zeros(1, 4, 576), torch.zeros(1, 4, 512, dtype=BF), torch.zeros(4, 576, dtype=BF)):
        with pytest.raises(RuntimeError, match="window"):
            kv4._window("x", kv, 576)
    with pytest.raises(RuntimeError, match="rope"):
        kv4._angles("x", torch.zeros(4, 31), torch.zeros(4, 31), 64, -1)


def test_entry_points_refuse():
    """Arguments that the C entry points turn away before any launch (addresses are never followed there)."""
    L, P, inv = _lib.lib(), 1 << 20, 1
    ok = dict(table=P, slots=2, cols=3, refs=P, pages=4, page=16, err=P)

    def pages(**k):
        d = {**ok, **k}
        return d["table"], d["slots"], d["cols"], d["refs"], d["pages"], d["page"], d["err"]
    for k in (dict(table=None), dict(slots=0), dict(cols=0), dict(refs=None), dict(pages=0), dict(page=48), dict(page=8),
              dict(page=512), dict(err=None), dict(slots=1 << 20, cols=1 << 12), dict(cols=256 * 65535 + 1, slots=1)):
        assert L.dsv41_kv4_fork(P, P, None, 1, *pages(**k), None) == inv, k
        assert L.dsv41_kv4_release(P, None, 1, *pages(**k), None) == inv, k
    assert L.dsv41_kv4_fork(None, P, None, 1, *pages(), None) == inv
    assert L.dsv41_kv4_fork(P, P, None, -1, *pages(), None) == inv
    assert L.dsv41_kv4_fork(None, None, None, 0, *pages(), None) == 0
    assert L.dsv41_kv4_release(None, None, 1, *pages(), None) == inv
    need = L.dsv41_kv4_reserve_workspace_bytes(5, 2, 4)
    assert need == 4 * (2 + 12 + 10)
    for n, pool, dim, ws, size in [(4097, P, 512, P, 1 << 30), (1, None, 512, P, need), (1, P + 8, 512, P, need),
                                   (1, P, 128, P, need), (5, P, 512, None, need), (5, P, 512, P, need - 1)]:
        assert L.dsv41_kv4_reserve(P, P, P, n, pool, dim, *pages(), ws, size, None) == inv
    assert L.dsv41_kv4_compact(P, 512, P, 2, 3, P, 4, 16, None, P, 1 << 20, None) == inv
    assert L.dsv41_kv4_compact(P, 512, P, 2, 3, P, 4, 16, P, P, L.dsv41_kv4_compact_workspace_bytes(4) - 1, None) == inv
    assert L.dsv41_kv4_copy_workspace_bytes(10, 100) == 0 and L.dsv41_kv4_copy_workspace_bytes(5000, 100) == 400
    assert L.dsv41_kv4_copy(P, 4, P + 512, 4, 16, 512, P, P, 1, P, None, 0, None) == inv  # (one memory)
    assert L.dsv41_kv4_copy(P, 4, 1 << 30, 4, 16, 512, P, P, 5000, P, None, 0, None) == inv
    for x, stride, ratio, rd, dim in [(None, 512, 4, 64, 512), (P + 2, 512, 4, 64, 512), (P, 500, 4, 64, 512),
                                      (P, 516, 4, 64, 512), (P, 512, 0, 64, 512), (P, 512, 4, 65, 512), (P, 640, 4, 64, 640)]:
        assert L.dsv41_kv4_append(x, stride, P, P, 1, ratio, P, P, 9, rd, P, 4, 16, dim, P, 2, 3, P, P, None) == inv
    assert L.dsv41_kv4_read(P, 4, 16, 512, P, 2, 3, P, P, 1, P + 2, None) == inv
    args = [P, P, 128 * 512, 2, 128, P, 4, 16, 512, P, 2, 3, P, 10, P, P, P, None, P, P, P, 100, 64, 1.0, P, 1, 16, None, 0, None]
    for at, v in [(0, None), (0, P + 2), (1, None), (4, 0), (5, None), (8, 256), (7, 20), (14, None), (15, None), (16, None),
                  (18, None), (19, None), (22, 62), (22, 516), (24, None), (26, 0), (13, -1), (2, 12)]:
        bad = list(args)
        bad[at] = v
        assert L.dsv41_sattn4(*bad) == inv, (at, v)
    # a workspace too small for the splits of one row over many keys
    bad = list(args)
    bad[13] = 4096
    assert L.dsv41_kv4_attn_workspace_bytes(1, 16, 128, 4096, 512, 0) > 0 and L.dsv41_sattn4(*bad) == inv
    args = [P, P, 128 * 512, 128, P, 128, P, 4, 16, 512, P, 2, 3, P, 10, None, P, 1.0, P, 1, 1, 16, None, 0, None]
    for at, v in [(0, None), (1, None), (4, None), (5, -1), (3, -1), (6, None), (13, None), (14, -1), (16, None), (18, None),
                  (21, 0)]:
        bad = list(args)
        bad[at] = v
        assert L.dsv41_sparse_attn4(*bad) == inv, (at, v)


def test_grid_is_the_reference_grid():
    """The tests' 4-bit grid is the oracle's fake quantisation (e4m3 scale), value for value, and its codes stand for it."""
    from oracle import dsv41_oracle as O
    rng = np.random.default_rng(0)
    x = O.bf16(rng.standard_normal((64, 576)).astype(np.float32) * np.exp2(rng.integers(-14, 12, (64, 1))).astype(np.float32))
    v, c, s = R.grid(torch.from_numpy(x).double())
    want = O.fake_quant_fp4(x, 16, scale_e4m3=True)
    big = np.abs(x).reshape(64, 36, 16).max(-1) > 2688  # (the oracle's scale there is the same, 448)
    assert np.array_equal(v.numpy().astype(np.float32), want), big.any()
    lut = torch.tensor(R.E2M1 + [-e for e in R.E2M1], dtype=torch.float64)
    assert torch.equal(lut[c.long()] * s.view(torch.float8_e4m3fn).double().repeat_interleave(16, 1), v)
    assert R.pack(torch.from_numpy(x).double()).shape == (64, 336)


def test_model_of_pages():
    m = R.Model(6, 3, 4, 16)
    assert m.reserve([0, 1], [0, 0], [17, 16]) and m.table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4]
    m.fork([0], [2], [17])
    assert m.refs().tolist() == [2, 2, 1, 0, 0, 0]
    assert m.reserve([2], [17], [18]) and m.table[2].tolist() == [0, 3, -1, -1]
    m.release([0], [0])
    assert m.compact() == 3 and m.table[2].tolist() == [0, 1, -1, -1] and m.table[1, 0] == 2
    assert not m.reserve([0], [0], [64])
