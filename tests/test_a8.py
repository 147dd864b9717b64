"""8-bit activations without a GPU: the container, the refusals of the shims and of the C entry points."""
import pytest
import torch

from dsv41_amd import A8, GatedFeedForward, gated_a8, linear_a8, norm_quant8
from dsv41_amd._lib import lib
from dsv41_amd.w8 import W8

import _a8_ref as R


def _a8(rows, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(rows, k, generator=g, dtype=torch.float64)
    codes, s = R.quantised(y)
    return A8(R.permuted(codes), R.pack_scales(s))


def _w8(n, k):
    return W8(torch.zeros(n, k, dtype=torch.uint8), torch.full(((n + 31) // 32, k // 32), 127, dtype=torch.uint8))


@pytest.mark.parametrize("k", [32, 96, 128, 160, 512])
def test_container_values(k):
    q = _a8(5, k)
    assert q.shape == (5, k) and q.s8.shape == ((k + 127) // 128, 5, 4)
    v = R.a8_values(q.a8, q.s8)
    assert torch.equal(q.float().double(), v) and torch.equal(q.bf16().double(), v)
    assert torch.equal(q.scales(), R.unpack_scales(q.s8, k))


def test_container_keeps_leading_sizes_and_nan_blocks():
    q = _a8(6, 64)
    q.s8[0, 2, 1] = 255
    r = A8(q.a8, q.s8, (2, 3, 64))
    v = r.float()
    assert v.shape == (2, 3, 64) and v[0, 2, 32:].isnan().all() and v.isnan().sum() == 32


def test_container_refusals():
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for a, s in [(u(4, 40), u(1, 4, 4)), (u(4, 64), u(4, 2)), (u(4, 64), u(2, 4, 4)), (u(4, 64).float(), u(1, 4, 4)),
                 (u(64), u(1, 1, 4)), (u(4, 64), u(1, 4, 4).int())]:
        with pytest.raises(ValueError):
            A8(a, s)
    for shape in [(4, 32), (2, 3, 64), (64,), (4, 2, 64)]:
        with pytest.raises(ValueError):
            A8(u(4, 64), u(1, 4, 4), shape)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        norm_quant8(x, x[0], 1e-6)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_a8(_a8(2, 64), _w8(32, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        gated_a8(_a8(2, 64), _w8(32, 64), _w8(32, 64))
    with pytest.raises(TypeError):
        linear_a8(x, _w8(32, 64))
    with pytest.raises(TypeError):
        linear_a8(_a8(2, 64), x)


def test_feed_forward_refuses_sizes_that_do_not_fit():
    n = torch.ones(64)
    GatedFeedForward(n, _w8(96, 64), _w8(96, 64), _w8(64, 96))
    for bad in [(n, _w8(96, 64), _w8(32, 64), _w8(64, 96)), (n, _w8(96, 64), _w8(96, 64), _w8(96, 64)),
                (n[:32], _w8(96, 64), _w8(96, 64), _w8(64, 96)), (n, _w8(100, 64), _w8(100, 64), _w8(64, 100 // 32 * 32))]:
        with pytest.raises(ValueError):
            GatedFeedForward(*bad)
    with pytest.raises(ValueError):
        GatedFeedForward(n, _w8(96, 64), _w8(96, 64), _w8(64, 96), act="swish")


# Addresses are never read by a refused call: any aligned number will do.
P = 1 << 20


def _norm(x=P, r=None, w=P, h=None, a8=P, s8=P, rows=4, D=64):
    return lib().dsv41_norm_quant8(x, r, w, 1e-6, h, a8, s8, rows, D, None)


def test_norm_entry_refusals():
    assert _norm(rows=0) == 0
    for bad in [dict(D=0), dict(D=48), dict(D=16416), dict(D=-32), dict(x=P + 8), dict(w=P + 2), dict(a8=P + 4),
                dict(x=None), dict(a8=None), dict(s8=None), dict(r=P), dict(r=P + 8, h=P), dict(r=P, h=P + 2), dict(rows=1 << 40)]:
        assert _norm(**bad) == 1, bad


def _linear(x=P, xs=P, w=P, ws=P, M=4, N=64, K=64, Kc=2, bias=None, bf=0, act=0, res=None, out=P, oa=None, os=None):
    return lib().dsv41_linear_a8(x, xs, w, ws, M, N, K, Kc, bias, bf, act, res, out, oa, os, None)


def _gated(x=P, xs=P, g=P, gs=P, u=P, us=P, M=4, N=64, K=64, Kg=2, Ku=2, act=2, limit=0.0, out=P, oa=None, os=None):
    return lib().dsv41_gated_a8(x, xs, g, gs, u, us, M, N, K, Kg, Ku, act, limit, out, oa, os, None)


def test_product_entry_refusals():
    for f in (_linear, _gated):
        assert f(M=0) == 0 and f(N=0) == 0
        for bad in [dict(M=-1), dict(N=-1), dict(M=0x7fffff01), dict(N=0x7fffff01), dict(x=None), dict(xs=None), dict(K=0), dict(K=48), dict(K=32800, Kc=1025) if f is _linear else dict(K=32800, Kg=1025, Ku=1025), dict(x=P + 8), dict(xs=P + 1), dict(act=5),
                    dict(act=-1), dict(out=None), dict(out=None, oa=P), dict(out=None, oa=P, os=P, N=40),
                    dict(out=None, oa=P + 8, os=P)]:
            assert f(**bad) == 1, (f.__name__, bad)
    for bad in [dict(w=P + 8), dict(w=None), dict(ws=None), dict(Kc=1)]:
        assert _linear(**bad) == 1, bad
    for bad in [dict(g=P + 8), dict(u=P + 8), dict(g=None), dict(gs=None), dict(u=None), dict(us=None), dict(Kg=1), dict(Ku=1), dict(limit=-1.0),
                dict(limit=float("nan"))]:
        assert _gated(**bad) == 1, bad


def test_products_of_more_rows_than_a_grid_holds():
    """A stream's row blocks are a grid's second size, at most 65535: more go to the tiles, and where K keeps them out the
    call is refused; so is one of more threads than a launch has."""
    plan = lib().dsv41_a8_plan
    for gated in (0, 1):
        for rows in (65535 * 64 + 1, 5000000, 1 << 26):
            assert plan(rows, 32, 32, gated, 0, 0) >> 30 == 1
        assert plan(65535 * 32 + 1, 32, 20000, gated, 0, 0) >> 16 in (48, 64)
    assert _linear(M=65535 * 64 + 1, K=20000, Kc=625) == 1
    assert _gated(M=65535 * 64 + 1, K=20000, Kg=625, Ku=625) == 1
    assert _linear(M=1 << 30, N=4096) == 1 and _linear(N=1 << 30) == 1


def test_counts_past_32_bits_are_refused():
    rows = (1 << 32) + 4
    meta = lambda *s: torch.empty(*s, dtype=torch.uint8, device="meta")  # noqa: E731
    x = A8(meta(rows, 64), meta(1, rows, 4))
    with pytest.raises(RuntimeError, match="at most"):
        linear_a8(x, _w8(32, 64))
    with pytest.raises(RuntimeError, match="at most"):
        gated_a8(x, _w8(32, 64), _w8(32, 64))
    with pytest.raises(ValueError):
        A8(meta(1, 64), meta(1, 1, 4), ())
