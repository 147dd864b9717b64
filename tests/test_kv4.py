"""The paged 4-bit cache on the CPU: what its calls refuse, workspace sizes, and the tests' own 64-bit forms."""
import ctypes

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
    c._pool, c._table, c._refs = _tensors(dim=dim)
    c.dim, c.pages, c.page, c.slots, c.cols, c.device, c.index = dim, 4, 16, 2, 3, torch.device("cpu"), -1
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
        c._i64("x", torch.zeros(3), 2)
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


def _struct(**k):
    P = 1 << 20
    return kv4._Cache(**{**dict(pool=P, table=P, refs=P, err=P, pages=4, page=16, slots=2, cols=3, dim=512), **k})


BAD_CACHES = [dict(pool=None), dict(pool=(1 << 20) + 8), dict(table=None), dict(refs=None), dict(err=None), dict(slots=0),
              dict(cols=0), dict(pages=0), dict(page=48), dict(page=8), dict(page=512), dict(dim=128), dict(dim=640),
              dict(slots=1 << 20, cols=1 << 12), dict(pages=1 << 27)]


def test_entry_points_refuse():
    """Arguments that the C entry points turn away before any launch (addresses are never followed there)."""
    L, P, inv = _lib.lib(), 1 << 20, 1
    c = ctypes.byref(_struct())
    big = 1 << 40
    for k in BAD_CACHES:
        x = ctypes.byref(_struct(**k))
        assert L.dsv41_kv4_fork(x, P, P, None, 1, None) == inv, k
        assert L.dsv41_kv4_release(x, P, None, 1, None) == inv, k
        assert L.dsv41_kv4_reserve(x, P, P, P, 1, P, big, None) == inv, k
        assert L.dsv41_kv4_compact(x, P, P, big, None) == inv, k
        assert L.dsv41_kv4_copy(x, ctypes.byref(_struct(pool=1 << 40)), P, P, 1, None, 0, None) == inv, k
        assert L.dsv41_kv4_copy(ctypes.byref(_struct(pool=1 << 40)), x, P, P, 1, None, 0, None) == inv, k
        assert L.dsv41_kv4_append(x, P, 1024, P, P, 1, 4, 0, P, P, 9, 64, None) == inv, k
        assert L.dsv41_kv4_read(x, P, P, 1, P, None) == inv, k
        assert L.dsv41_sattn4(x, P, P, 128 * 512, 2, 128, P, 10, P, P, P, None, P, P, P, 100, 64, 1.0, P, 1, 16, None, 0, None) == inv
        assert L.dsv41_sparse_attn4(x, P, P, 128 * 512, 128, P, 128, P, 10, None, P, 1.0, P, 1, 1, 16, None, 0, None) == inv
    assert L.dsv41_kv4_fork(None, P, P, None, 1, None) == inv
    wide = ctypes.byref(_struct(slots=1, cols=256 * 65535 + 1))
    assert L.dsv41_kv4_fork(wide, P, P, None, 1, None) == inv and L.dsv41_kv4_release(wide, P, None, 1, None) == inv
    assert L.dsv41_kv4_fork(c, None, P, None, 1, None) == inv and L.dsv41_kv4_fork(c, P, None, None, 1, None) == inv
    assert L.dsv41_kv4_fork(c, P, P, None, -1, None) == inv and L.dsv41_kv4_fork(c, None, None, None, 0, None) == 0
    assert L.dsv41_kv4_release(c, None, None, 1, None) == inv
    need = L.dsv41_kv4_reserve_workspace_bytes(c, 5)
    assert need == 4 * (2 + 12 + 10)
    for n, ws, size in [(4097, P, big), (-1, P, big), (5, None, need), (5, P + 2, need), (5, P, need - 1)]:
        assert L.dsv41_kv4_reserve(c, P, P, P, n, ws, size, None) == inv
    need = L.dsv41_kv4_compact_workspace_bytes(c)
    assert need == 4 * 14
    assert L.dsv41_kv4_compact(c, None, P, big, None) == inv and L.dsv41_kv4_compact(c, P, P, need - 1, None) == inv
    assert L.dsv41_kv4_copy_workspace_bytes(c, 10) == 0 and L.dsv41_kv4_copy_workspace_bytes(c, 50000) == 16
    assert L.dsv41_kv4_copy(c, ctypes.byref(_struct(pool=P + 512)), P, P, 1, None, 0, None) == inv  # (one memory)
    far = dict(pool=1 << 40)
    assert L.dsv41_kv4_copy(c, ctypes.byref(_struct(**far)), P, P, 50000, None, 0, None) == inv
    assert L.dsv41_kv4_copy(c, ctypes.byref(_struct(**far, page=32)), P, P, 1, None, 0, None) == inv
    assert L.dsv41_kv4_copy(c, ctypes.byref(_struct(**far, dim=576)), P, P, 1, None, 0, None) == inv
    for x, stride, ratio, rd in [(None, 512, 4, 64), (P + 2, 512, 4, 64), (P, 500, 4, 64), (P, 516, 4, 64), (P, 512, 0, 64),
                                 (P, 512, 4, 65), (P, 512, 4, 514), (P, 512, 4, -2)]:
        assert L.dsv41_kv4_append(c, x, stride, P, P, 1, ratio, 0, P, P, 9, rd, None) == inv
    assert L.dsv41_kv4_append(c, P, 512, P, P, 1, 4, 1, None, P, 9, 64, None) == inv
    assert L.dsv41_kv4_read(c, P, P, 1, P + 2, None) == inv
    args = [c, P, P, 128 * 512, 2, 128, P, 10, P, P, P, None, P, P, P, 100, 64, 1.0, P, 1, 16, None, 0, None]
    for at, v in [(1, None), (1, P + 2), (2, None), (3, 12), (5, 0), (6, None), (7, -1), (8, None), (9, None), (10, None),
                  (12, None), (13, None), (16, 62), (16, 516), (16, -4), (18, None), (18, P + 8), (19, -1), (20, 0), (5, 0x7fffffff),
                  (7, 0x7fffffff)]:
        bad = list(args)
        bad[at] = v
        assert L.dsv41_sattn4(*bad) == inv, (at, v)
    # a workspace too small for the splits of one row over many keys
    bad = list(args)
    bad[7] = 4096
    assert L.dsv41_kv4_attn_workspace_bytes(c, 1, 16, 128, 4096, 0) > 0 and L.dsv41_sattn4(*bad) == inv
    args = [c, P, P, 128 * 512, 128, P, 128, P, 10, None, P, 1.0, P, 1, 1, 16, None, 0, None]
    for at, v in [(1, None), (2, None), (4, -1), (5, None), (6, -1), (7, None), (8, -1), (10, None), (12, None), (13, -1),
                  (14, -1), (15, 0), (4, 0x7fffffff), (6, 0x7fffffff), (8, 0x7fffffff), (12, P + 8)]:
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


def test_workspace_sizes_agree():
    """The sizes that the Python calls allocate are those that the library asks for."""
    from dsv41_amd import kv4
    L = _lib.lib()
    s = _struct(pages=700, slots=9, cols=11)
    c = ctypes.byref(s)
    for n in (1, 4, 5, kv4._MOST_ENTRIES):
        assert L.dsv41_kv4_reserve_workspace_bytes(c, n) == 4 * (9 + 3 * 700 + 2 * n)
    assert L.dsv41_kv4_compact_workspace_bytes(c) == 4 * (2 + 3 * 700)
    assert L.dsv41_kv4_copy_workspace_bytes(c, kv4._FEW_COPIES) == 0
    assert L.dsv41_kv4_copy_workspace_bytes(c, kv4._FEW_COPIES + 1) == 4 * 700
