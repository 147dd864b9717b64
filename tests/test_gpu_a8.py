"""Parity of the 8-bit activation operators with their 64-bit reference (tests/_a8_ref.py).

Tolerances.  Products of small whole numbers have sums that fp32 and the matrix instructions hold exactly, so outputs are
compared bit for bit with the once-rounded sum: every k, row, column and scale has to be in its place.  For other inputs:
the matrix instructions add the products of an instruction with an error of at most 2^-11 of the sum of their magnitudes
(measured 2^-11.6 at worst over codes of every exponent; 2^-16 of the result in the 2-norm of random ones), an activation
adds at most 2e-5 relative (e^z of a z that is off by 3 roundings of 2^-24 is off by 3 |z| 2^-24, |z| <= 88 before it is 0
or infinite: 1.6e-5; the other factors under 16 roundings), and the result is rounded by half a step (bf16 2^-8 relative at most, 2^-8 / sqrt 3 in the
2-norm of many; e4m3 2^-4)."""
import zlib

import pytest
import torch

import _a8_ref as R
from dsv41_amd import A8, GatedFeedForward, gated_a8, linear_a8, norm_quant8
from dsv41_amd.w8 import W8

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda:0"
EPS = 1e-6
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
SUM_ERR, ACT_ERR = 2.0 ** -11, 2e-5


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


# ------------------------------------------------------------------------------------------------ inputs
def random_a8(g, rows, k, wide=False):
    """Quantised normal rows, a few channels far larger (wide: codes and scales of every size)."""
    if wide:
        codes = torch.randint(0, 256, (rows, k), generator=g).to(torch.uint8)
        codes[(codes & 127) == 127] = 1
        s = torch.randint(121, 129, (rows, k // 32), generator=g).to(torch.uint8)
    else:
        y = torch.randn(rows, k, generator=g, dtype=torch.float64)
        y[:, ::97] *= 20
        codes, s = R.quantised(y)
    return A8(R.permuted(codes).to(DEV), R.pack_scales(s).to(DEV)), R.a8_values(R.permuted(codes), R.pack_scales(s))


def whole_a8(g, rows, k):
    """Whole numbers -2 .. 2 times 2^-1 .. 2^1 per block."""
    codes = torch.tensor([0x00, 0x38, 0x40, 0xb8, 0xc0], dtype=torch.uint8)[torch.randint(0, 5, (rows, k), generator=g)]
    s = torch.randint(126, 129, (rows, k // 32), generator=g).to(torch.uint8)
    return A8(R.permuted(codes).to(DEV), R.pack_scales(s).to(DEV)), R.a8_values(R.permuted(codes), R.pack_scales(s))


def random_w8(g, n, k):
    nb = -(-n // 32)
    y = torch.randn(nb * 32, k, generator=g, dtype=torch.float64) * k ** -0.5
    a = y.view(nb, 32, k // 32, 32).abs().amax((1, 3))
    s = (torch.ceil(torch.log2(a / 448)) + 127).to(torch.uint8)
    v = y / R.scale_values(s).repeat_interleave(32, 0).repeat_interleave(32, 1)
    codes = v.float().to(torch.float8_e4m3fn).view(torch.uint8)[:n].contiguous()
    return W8(codes.to(DEV), s.to(DEV)), R.w8_values(codes, s)


def whole_w8(g, n, k):
    codes = torch.tensor([0x00, 0x38, 0x40, 0xb8, 0xc0], dtype=torch.uint8)[torch.randint(0, 5, (n, k), generator=g)]
    s = torch.randint(126, 129, (-(-n // 32), k // 32), generator=g).to(torch.uint8)
    return W8(codes.to(DEV), s.to(DEV)), R.w8_values(codes, s)


def bf(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF)


# ------------------------------------------------------------------------------------------------ comparisons
def check_a8(q, want, err):
    """q (A8) against float64 rows `want`, known to `err` each: the block's scale unless the largest value is within err
    of a power of two's border, every value within half a step of the scale it has."""
    want, err = want.reshape(-1, want.shape[-1]), err.reshape(-1, want.shape[-1])
    rows, k = want.shape
    assert q.a8.shape == (rows, k)
    s8 = q.s8.cpu()
    pad = s8.permute(1, 0, 2).reshape(rows, -1)[:, k // 32:]
    assert (pad == 127).all()
    s = R.unpack_scales(s8, k).double() - 127
    b = want.view(rows, -1, 32).abs()
    lo = R.block_exponents((b - err.view(rows, -1, 32)).clamp_min(0).reshape(rows, k))
    hi = R.block_exponents((b + err.view(rows, -1, 32)).reshape(rows, k))
    assert ((s >= lo) & (s <= hi)).all(), "scales"
    sv = (2.0 ** s).repeat_interleave(32, 1)
    got = R.a8_values(q.a8.cpu(), s8)
    off = (got - want).abs()
    tol = R.half_steps(((want.abs() + err) / sv).clamp_max(448)) * sv + err
    assert (off <= tol).all(), (off / tol).max()


def check_bf16(y, want, err):
    got = y.double().cpu().view(want.shape)
    off = (got - want).abs()
    tol = err + (want.abs() + err) * 2.0 ** -8
    assert (off <= tol).all(), (off / tol).max()
    rms = lambda t: t.pow(2).mean().sqrt()  # noqa: E731
    if off.numel() >= 1024:
        assert rms(off) <= 1.05 * 2.0 ** -8 / 3 ** 0.5 * rms(want) + rms(err) / 16, "2-norm"


# ------------------------------------------------------------------------------------------------ norm_quant8
@pytest.mark.parametrize("rows,d", [(1, 32), (3, 64), (5, 160), (1, 512), (7, 544), (4, 1024), (9, 1280), (2, 2048),
                                    (3, 2080), (1, 5120), (6, 5120), (2, 8192), (3, 8224), (2, 16384)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_norm_quant8(rows, d, residual, norm):
    g = gen("norm", rows, d, residual, norm)
    x, r, w = bf(g, rows, d), bf(g, rows, d, scale=5.0), (torch.rand(d, generator=g) + 0.5).to(BF)
    x[:, ::53] *= 30
    out = norm_quant8(x.to(DEV), w.to(DEV) if norm else None, EPS, residual=r.to(DEV) if residual else None)
    h = x
    if residual:
        out, hg = out
        h = (x.float() + r.float()).to(BF)
        assert torch.equal(hg.cpu(), h)
    assert out.shape == (rows, d)
    y = R.normed(h.double(), w.double(), EPS) if norm else h.double()
    # fp32: the sum of squares, its root and quotient, two products: under 16 roundings of 2^-24
    check_a8(out, y, y.abs() * 16 * 2.0 ** -24 if norm else torch.zeros_like(y))


def test_norm_quant8_is_the_grid_of_fake_quant():
    from dsv41_amd.fused import fake_quant_fp8
    g = gen("grid")
    x = bf(g, 37, 1280, scale=3.0)
    x[3] = 0
    x[4, :32] = 1e-9
    x[5] *= 1e30
    q = norm_quant8(x.to(DEV), None, 0.0)
    assert torch.equal(q.bf16(), fake_quant_fp8(x.to(DEV)))


def test_norm_quant8_rows_without_a_number():
    """Infinities and NaN: a block that holds one is NaN; zero rows are zero; other rows are untouched."""
    g = gen("nan")
    for d in (1280, 5120):
        x = bf(g, 6, d)
        x[1, 40], x[2, 7], x[4] = float("inf"), float("nan"), 0
        ones = torch.ones(d, dtype=BF)
        q = norm_quant8(x.to(DEV), None, 0.0)
        v = q.float().cpu()
        assert v[1, 32:64].isnan().all() and v[1, 64:].isfinite().all() and v[1, :32].isfinite().all()
        assert v[2, :32].isnan().all() and v[2, 32:].isfinite().all()
        assert (q.scales().cpu()[1] == 255).nonzero().flatten().tolist() == [1]
        q = norm_quant8(x.to(DEV), ones.to(DEV), EPS)
        v = q.float().cpu()
        assert v[1, 32:64].isnan().all() and (v[1, 64:] == 0).all()  # 1 / inf, and inf * 0
        assert v[2].isnan().all() and (v[4] == 0).all()
        keep = [0, 3, 5]
        check_a8(A8(q.a8[keep], q.s8[:, keep]), R.normed(x[keep].double(), ones.double(), EPS),
                 R.normed(x[keep].double(), ones.double(), EPS).abs() * 2.0 ** -20)


def test_norm_quant8_views_and_sizes():
    g = gen("views")
    base = bf(g, 8, 3, 1300)
    x = base.to(DEV)[:, ::2, 4:1284]  # strided, not 16-byte aligned
    r = bf(g, 8, 2, 1280).to(DEV)
    w = (torch.rand(1281, generator=g) + 0.5).to(BF).to(DEV)[1:]
    q, h = norm_quant8(x, w, EPS, residual=r)
    q2, h2 = norm_quant8(x.contiguous(), w.clone(), EPS, residual=r)
    assert q.shape == (8, 2, 1280) and torch.equal(h, h2) and torch.equal(q.a8, q2.a8) and torch.equal(q.s8, q2.s8)
    qf = norm_quant8(x, w.float(), EPS)
    assert torch.equal(qf.a8, norm_quant8(x, w, EPS).a8)
    e, he = norm_quant8(x[:0], w, EPS, residual=r[:0])
    assert e.shape == (0, 2, 1280) and e.a8.shape == (0, 1280) and he.shape == (0, 2, 1280)


# ------------------------------------------------------------------------------------------------ linear_a8
SIZES = [(1, 1, 32), (1, 33, 64), (2, 100, 96), (5, 512, 128), (15, 257, 160), (16, 64, 1280), (17, 96, 1312), (31, 130, 224),
         (32, 2080, 512), (33, 64, 32), (40, 129, 96), (64, 257, 1280), (65, 1000, 160), (127, 128, 2080), (129, 384, 640),
         (200, 511, 5120), (257, 260, 352), (300, 1280, 288)]
LARGE = [(2049, 513, 288), (2100, 1056, 1184), (4097, 256, 128), (1, 16416, 128), (20, 17000, 160), (3, 4096, 8224),
         (30, 2080, 4128), (1100, 2080, 160), (450, 4640, 6176), (1024, 8160, 640), (2049, 4096, 1312), (4090, 4064, 1280),
         (70, 64, 20000), (40, 33, 32768), (2049, 7233, 160), (4090, 4928, 160)]


def plan(m, n, k, gated=False, a8=False, rest=False):
    from dsv41_amd._lib import lib
    return lib().dsv41_a8_plan(m, n, k, int(gated), int(a8), int(rest))


def test_sizes_reach_every_kernel():
    """(exact sums, tile, rows, columns, waves) of the streams and tiles that the sizes below run on."""
    kind = lambda m, p: (m <= 32, p >> 30, p >> 16 & 0x3fff, p >> 4 & 0xfff, p & 15)  # noqa: E731
    tiles = {(False, 1, *t) for t in ((128, 64, 4), (128, 128, 8), (256, 128, 8), (192, 256, 8), (256, 256, 8))}
    exact = {(True, 0, *t) for t in ((16, 16, 8), (16, 16, 4), (16, 32, 4), (16, 32, 2), (32, 32, 4), (32, 32, 2))}
    linear = {kind(s[0], plan(*s, a8=a)) for s in SIZES + LARGE for a in (False, True) if not a or s[1] % 32 == 0}
    assert linear == tiles | exact | {(True, 0, 32, 16, 4)} | {(False, 0, r, 32, 4) for r in (32, 48, 64)}
    gated = {kind(s[0], plan(*s, gated=True, a8=a)) for s in GATED + GATED_LARGE for a in (False, True)}
    assert gated == tiles | exact | {(False, 0, r, 64, 4) for r in (32, 48, 64)}
    for sizes, g in ((LARGE, False), (GATED_LARGE, True)):  # columns behind the last whole round on another kernel
        assert sum(plan(*s, gated=g, rest=True) != 0 for s in sizes) >= 2


@pytest.mark.parametrize("m,n,k", SIZES + LARGE)
def test_linear_a8_whole_numbers(m, n, k):
    g = gen("whole", m, n, k)
    (x, xv), (w, wv) = whole_a8(g, m, k), whole_w8(g, n, k)
    y = linear_a8(x, w)
    want = (xv.to(DEV) @ wv.to(DEV).t()).cpu()
    assert y.shape == (m, n) and y.dtype == BF and torch.equal(y.cpu(), want.to(BF))
    if n % 32 == 0:
        q = linear_a8(x, w, out=A8)
        check_a8(q, want, torch.zeros_like(want))
        assert torch.equal(q.a8, linear_a8(x, w, out=A8).a8)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("wide", [False, True])
def test_linear_a8(m, n, k, wide):
    g = gen("linear", m, n, k, wide)
    (x, xv), (w, wv) = random_a8(g, m, k, wide), random_w8(g, n, k)
    want = xv @ wv.t()
    check_bf16(linear_a8(x, w), want, (xv.abs() @ wv.abs().t()) * SUM_ERR)


@pytest.mark.parametrize("m,n,k", [(1, 100, 256), (3, 128, 5120), (20, 96, 640), (48, 130, 320), (150, 64, 2048),
                                   (300, 513, 160), (2300, 260, 96)])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [None, BF, torch.float32])
def test_linear_a8_epilogue(m, n, k, act, bias):
    g = gen("epi", m, n, k, act, str(bias))
    (x, xv), (w, wv) = whole_a8(g, m, k), whole_w8(g, n, k)
    w = W8(w.w8, w.s8 - 6, permuted=True)  # (sums of a size at which the activations bend)
    pre = xv @ wv.t() / 64
    b = None
    if bias is not None:
        b = torch.randn(n, generator=g).to(bias)
        pre = (pre.float() + b.float()).double()  # (exact sums, one fp32 addition)
    r = bf(g, m, n)
    y0 = R.act(pre, act)
    kw = dict(bias=None if b is None else b.to(DEV), act=act)
    check_bf16(linear_a8(x, w, **kw), y0, y0.abs() * ACT_ERR + 1e-30)
    y1 = y0 + r.double()
    check_bf16(linear_a8(x, w, residual=r.to(DEV), **kw), y1, y0.abs() * ACT_ERR + y1.abs() * 2.0 ** -23 + 1e-30)
    if n % 32 == 0:
        check_a8(linear_a8(x, w, out=A8, **kw), y0, y0.abs() * ACT_ERR + 1e-30)


@pytest.mark.parametrize("act", ACTS[1:])
def test_activations_over_their_range(act):
    """One product per output: sums from -448 * 2^k to 448 * 2^k through x = each code, w = 1, scales 2^-12 .. 2^3."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 127) != 127]
    xs = torch.zeros(len(codes) * 16, 32, dtype=torch.uint8)
    xs[:, 0] = codes.repeat(16)
    s = (torch.arange(16) + 115).repeat_interleave(len(codes)).to(torch.uint8).unsqueeze(1)
    x, xv = A8(R.permuted(xs).to(DEV), R.pack_scales(s).to(DEV)), R.a8_values(R.permuted(xs), R.pack_scales(s))
    w = torch.zeros(4, 32, dtype=torch.uint8)
    w[:, 0] = 0x38
    y = linear_a8(x, W8(w.to(DEV), torch.full((1, 1), 127, dtype=torch.uint8, device=DEV)), act=act)
    want = R.act(xv[:, :1].expand(-1, 4).contiguous(), act)
    off = (y.cpu().double() - want).abs()
    tiny = 2.0 ** -126 * (1 + xv[:, :1].abs())  # (factors and results under the smallest normal number may be flushed)
    assert (off <= want.abs() * (2.0 ** -8 + 2e-5) + tiny).all(), (off / (want.abs() + tiny)).max()


@pytest.mark.parametrize("m", [1, 20, 50, 130, 2200])
def test_linear_a8_without_a_number(m):
    """NaN blocks of x make their rows NaN and no other row; infinite bias and residual pass through."""
    g = gen("nan", m)
    (x, xv), (w, wv) = whole_a8(g, m, 320), whole_w8(g, 96, 320)
    x.s8[2, m // 2, 1] = 255
    y = linear_a8(x, w)
    want = xv @ wv.t()
    want[m // 2] = float("nan")
    assert torch.equal(y.cpu().nan_to_num(7777.0), want.to(BF).nan_to_num(7777.0))
    q = linear_a8(x, w, out=A8)
    assert (q.scales()[m // 2] == 255).all() and q.float()[m // 2].isnan().all() and q.float().isnan().sum() == 96
    x.s8[2, m // 2, 1] = 127
    b = torch.zeros(96, device=DEV)
    b[5], b[6] = float("inf"), float("-inf")
    for act, lo in [("none", float("-inf")), ("relu", 0.0)]:
        y = linear_a8(x, w, bias=b, act=act).cpu().float()
        assert (y[:, 5] == float("inf")).all() and (y[:, 6] == lo).all() and y[:, 7:].isfinite().all()


def test_linear_a8_views_shapes_and_empty():
    g = gen("lv")
    (x, xv), (w, wv) = whole_a8(g, 6, 256), whole_w8(g, 40, 256)
    want = (xv @ wv.t()).to(BF)
    x3 = A8(x.a8, x.s8, (2, 3, 256))
    r = torch.zeros(3, 2, 40, dtype=BF, device=DEV).transpose(0, 1)
    assert torch.equal(linear_a8(x3, w, residual=r).cpu(), want.view(2, 3, 40))
    off = torch.empty(6 * 256 + 1, dtype=torch.uint8, device=DEV)[1:].view(6, 256)
    off.copy_(x.a8)
    so = torch.empty(x.s8.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(x.s8.shape)
    so.copy_(x.s8)
    wo = torch.empty(40 * 256 + 3, dtype=torch.uint8, device=DEV)[3:].view(40, 256)
    wo.copy_(w.w8)
    bo = torch.zeros(41, device=DEV, dtype=BF)[1:]
    assert torch.equal(linear_a8(A8(off, so), W8(wo, w.s8, permuted=True), bias=bo).cpu(), want)
    wide = torch.full((2, 20), 99, dtype=torch.uint8, device=DEV)  # scales of more columns than K has
    wide[:, :8] = w.s8
    assert torch.equal(linear_a8(x, W8(w.w8, wide, permuted=True)).cpu(), want)
    e = linear_a8(A8(x.a8[:0], x.s8[:, :0]), w)
    assert e.shape == (0, 40)
    assert linear_a8(A8(x.a8[:0], x.s8[:, :0]), whole_w8(g, 64, 256)[0], out=A8).a8.shape == (0, 64)


def test_refusals():
    g = gen("ref")
    (x, _), (w, _), (w2, _) = whole_a8(g, 4, 128), whole_w8(g, 64, 128), whole_w8(g, 40, 128)
    t = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    bad = [(ValueError, lambda: linear_a8(x, w, act="swish")), (ValueError, lambda: linear_a8(x, w, out=torch.float32)),
           (RuntimeError, lambda: linear_a8(x, whole_w8(g, 64, 96)[0])), (RuntimeError, lambda: linear_a8(x, w2, out=A8)),
           (RuntimeError, lambda: linear_a8(x, w, bias=t(63))), (RuntimeError, lambda: linear_a8(x, w, bias=t(64).half())),
           (RuntimeError, lambda: linear_a8(x, w, bias=t(64).cpu())), (RuntimeError, lambda: linear_a8(x, w, residual=t(64))),
           (RuntimeError, lambda: linear_a8(x, w, residual=t(4, 64, dt=torch.float32))),
           (RuntimeError, lambda: linear_a8(x, w, bias=t(64).requires_grad_())),
           (RuntimeError, lambda: linear_a8(x, W8(w.w8, w.s8[:1], permuted=True))),
           (RuntimeError, lambda: gated_a8(x, w, w2)), (ValueError, lambda: gated_a8(x, w, w, limit=-1.0)),
           (RuntimeError, lambda: gated_a8(x, w2, w2)), (RuntimeError, lambda: norm_quant8(t(2, 48), None, EPS)),
           (RuntimeError, lambda: norm_quant8(t(2, 16416), None, EPS)), (RuntimeError, lambda: norm_quant8(t(2, 64), t(32), EPS)),
           (RuntimeError, lambda: norm_quant8(t(2, 64), t(64), EPS, residual=t(64))),
           (RuntimeError, lambda: norm_quant8(t(2, 64).float(), t(64), EPS)),
           (RuntimeError, lambda: norm_quant8(t(2, 64), t(64).requires_grad_(), EPS))]
    for i, (err, f) in enumerate(bad):
        with pytest.raises(err):
            f()
            print("not refused:", i)
    with torch.no_grad():
        norm_quant8(t(2, 64), t(64).requires_grad_(), EPS)


# ------------------------------------------------------------------------------------------------ gated_a8
GATED = [(1, 32, 32), (2, 96, 96), (16, 512, 1280), (17, 64, 160), (32, 224, 512), (33, 32, 64), (64, 160, 1280),
         (100, 1024, 352), (140, 1952, 160), (200, 2016, 352), (129, 416, 5120), (300, 288, 160), (2049, 288, 224)]
GATED_LARGE = [(2, 16416, 96), (5, 2080, 4128), (18, 16896, 64), (1100, 1056, 160), (450, 2336, 6176), (1024, 4064, 640),
               (2049, 2048, 1312), (4090, 2016, 1280), (1100, 6560, 160), (4090, 2528, 160)]


@pytest.mark.parametrize("m,n,k", GATED)
@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("gelu_tanh", 0.75), ("gelu", 0.0), ("none", 0.5), ("relu", 0.0)])
def test_gated_a8(m, n, k, act, limit):
    g = gen("gated", m, n, k, act)
    (x, xv), (wg, gv), (wu, uv) = whole_a8(g, m, k), whole_w8(g, n, k), whole_w8(g, n, k)
    wg, wu = W8(wg.w8, wg.s8 - 5, permuted=True), W8(wu.w8, wu.s8 - 4, permuted=True)
    gate, up = xv @ gv.t() / 32, xv @ uv.t() / 16
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    want = R.act(gate, act) * up
    err = want.abs() * (ACT_ERR + 2.0 ** -23) + 1e-30
    y = gated_a8(x, wg, wu, act=act, limit=limit, out=BF)
    check_bf16(y, want, err)
    q = gated_a8(x, wg, wu, act=act, limit=limit)
    check_a8(q, want, err)
    again = gated_a8(x, wg, wu, act=act, limit=limit)
    assert torch.equal(q.a8, again.a8) and torch.equal(q.s8, again.s8)


@pytest.mark.parametrize("m,n,k", GATED_LARGE)
def test_gated_a8_large(m, n, k):
    g = gen("gated large", m, n, k)
    (x, xv), (wg, gv), (wu, uv) = whole_a8(g, m, k), whole_w8(g, n, k), whole_w8(g, n, k)
    wg, wu = W8(wg.w8, wg.s8 - 6, permuted=True), W8(wu.w8, wu.s8 - 4, permuted=True)
    gate, up = ((xv.to(DEV) @ v.to(DEV).t()).cpu() / d for v, d in ((gv, 64), (uv, 16)))
    want = R.act(gate, "silu") * up
    err = want.abs() * (ACT_ERR + 2.0 ** -23) + 1e-30
    check_bf16(gated_a8(x, wg, wu, out=BF), want, err)
    check_a8(gated_a8(x, wg, wu), want, err)


def test_gated_a8_odd_columns_in_bf16():
    g = gen("odd")
    for m in (3, 40, 140, 2100):
        (x, xv), (wg, gv), (wu, uv) = whole_a8(g, m, 96), whole_w8(g, 77, 96), whole_w8(g, 77, 96)
        want = torch.relu(xv @ gv.t()) * (xv @ uv.t())
        check_bf16(gated_a8(x, wg, wu, act="relu", out=BF), want, want.abs() * 2.0 ** -23)


def test_gated_a8_limit_lets_nan_pass():
    g = gen("gn")
    for m in (2, 40, 130):
        (x, _), (wg, _), (wu, _) = whole_a8(g, m, 128), whole_w8(g, 32, 128), whole_w8(g, 32, 128)
        x.s8[0, 1, 2] = 255
        v = gated_a8(x, wg, wu, limit=1.0).float()
        assert v[1].isnan().all() and v.isnan().sum() == 32


# ------------------------------------------------------------------------------------------------ together
def ffn_reference(x, r, norm, gv, uv, dv, limit):
    h = (x.float() + r.float()).to(BF)
    y = R.normed(h.double(), norm.double(), EPS)
    c, s = R.quantised(y)
    a = R.a8_values(R.permuted(c), R.pack_scales(s))
    gate, up = a @ gv.t(), a @ uv.t()
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    p = R.act(gate, "silu") * up
    c, s = R.quantised(p)
    b = R.a8_values(R.permuted(c), R.pack_scales(s))
    return h.double() + b @ dv.t(), p


@pytest.mark.parametrize("rows", [1, 6, 33, 150])
@pytest.mark.parametrize("limit", [0.0, 2.0])
def test_feed_forward(rows, limit):
    g = gen("ffn", rows, limit)
    dim, F = 640, 416
    norm = (torch.rand(dim, generator=g) + 0.5).to(BF)
    (wg, gv), (wu, uv), (wd, dv) = random_w8(g, F, dim), random_w8(g, F, dim), random_w8(g, dim, F)
    x, r = bf(g, 2, rows, dim), bf(g, 2, rows, dim, scale=2.0)
    f = GatedFeedForward(norm.to(DEV), wg, wu, wd, eps=EPS, limit=limit)
    y = f(x.to(DEV), residual=r.to(DEV))
    assert y.shape == (2, rows, dim)
    want, p = ffn_reference(x.view(-1, dim), r.view(-1, dim), norm, gv, uv, dv, limit)
    # single codes of the two quantisations may fall to the other side of a border: a step of 2^-3 of a value, at most a
    # thousandth of them (their inputs are off by 2^-16, a border lies within that of one value in 2^12)
    off = (y.double().cpu().view(want.shape) - want).abs()
    tol = want.abs() * 2.0 ** -8 + p.abs().amax(-1, keepdim=True) * dv.abs().amax() * 2.0 ** -3 * 4
    assert (off <= tol).all(), (off / tol).max()
    rms = lambda t: t.pow(2).mean().sqrt()  # noqa: E731
    part = want - (x.float() + r.float()).to(BF).double().view(want.shape)  # (codes off: 2^-3 * 2^-6 in the 2-norm, twice)
    assert rms(off) <= 1.05 * 2.0 ** -8 / 3 ** 0.5 * rms(want) + 2.0 ** -8 * rms(part)
    alone = f((x.float() + r.float()).to(BF).to(DEV))
    assert torch.equal(alone, y)


def test_feed_forward_captured_on_two_streams():
    """Two captured graphs and eager calls between their replays, on their own streams."""
    g = gen("cap")
    dim, F, rows = 512, 256, 70
    norm = torch.ones(dim, dtype=BF)
    f = [GatedFeedForward(norm.to(DEV), random_w8(g, F, dim)[0], random_w8(g, F, dim)[0], random_w8(g, dim, F)[0])
         for _ in range(2)]
    x = [bf(g, rows, dim).to(DEV) for _ in range(2)]
    r = [bf(g, rows, dim).to(DEV) for _ in range(2)]
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(side[i]):
            f[i](x[i], residual=r[i])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[i]):
            outs.append(f[i](x[i], residual=r[i]))
        graphs.append(graph)
    for rep in range(4):
        for i in range(2):
            x[i].copy_(bf(g, rows, dim))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        eager = [f[i](x[i], residual=r[i]) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager[i]), (rep, i)


def test_product_of_two_launches_captured():
    g = gen("two parts")
    m, n, k = 2049, 7232, 160
    assert plan(m, n, k, rest=True)
    (x, _), (w, _), (z, _) = random_a8(g, m, k), random_w8(g, n, k), random_a8(g, m, k)
    r = bf(g, m, n).to(DEV)
    linear_a8(x, w, residual=r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear_a8(x, w, residual=r)
        q = linear_a8(x, w, out=A8)
    for rep in range(3):
        if rep == 2:
            x.a8.copy_(z.a8)
            x.s8.copy_(z.s8)
        graph.replay()
        eager, codes = linear_a8(x, w, residual=r), linear_a8(x, w, out=A8)
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and torch.equal(q.a8, codes.a8) and torch.equal(q.s8, codes.s8), rep


def test_results_do_not_depend_on_other_rows():
    """A row's result is the same bits whatever rows stand beside it in the same kernel, and rows behind are left alone."""
    g = gen("rows")
    (x, _), (w, _) = random_a8(g, 300, 640), random_w8(g, 256, 640)
    y = linear_a8(x, w)
    z = linear_a8(A8(x.a8[7:], x.s8[:, 7:]), w)
    assert torch.equal(y[7:], z)
    y = linear_a8(A8(x.a8[:9], x.s8[:, :9]), w)
    z = linear_a8(A8(x.a8[8:9], x.s8[:, 8:9]), w)
    assert torch.equal(y[8:], z)


def test_offsets_past_32_bits():
    """Outputs and codes of more than 2^31 values: the last rows against the same rows alone."""
    g = gen("big")
    k, n, m = 64, 32768, 70001
    (x, _), (w, _) = whole_a8(g, 71, k), whole_w8(g, n, k)
    codes = torch.zeros(m, k, dtype=torch.uint8, device=DEV)
    scales = torch.full((1, m, 4), 127, dtype=torch.uint8, device=DEV)
    codes[-71:], scales[:, -71:] = x.a8, x.s8
    want = linear_a8(x, w)
    y = linear_a8(A8(codes, scales), w)
    assert torch.equal(y[-71:], want) and not y[:5].any()
    del y
    q = linear_a8(A8(codes, scales), w, out=A8)
    assert torch.equal(A8(q.a8[-71:], q.s8[:, -71:]).bf16(), linear_a8(x, w, out=A8).bf16())
    t = norm_quant8(torch.ones(70001, 1, dtype=BF, device=DEV).expand(-1, 32768)[:, :16384].contiguous(), None, 0.0)
    assert (t.s8 == 119).all() and (t.a8[-1] == 0x78).all()


@pytest.mark.parametrize("rows,d", [((1 << 25) + 5, 32), ((1 << 21) + 3, 2080)])
def test_norm_quant8_of_more_rows_than_a_launch_has(rows, d):
    """The rows of a second launch against the same rows alone."""
    g = gen("launches", d)
    x = torch.ones(rows, d, dtype=BF, device=DEV)
    x[-9:] = bf(g, 9, d).to(DEV)
    w = (torch.rand(d, generator=g) + 0.5).to(BF).to(DEV)
    q, last, first = norm_quant8(x, w, EPS), norm_quant8(x[-9:], w, EPS), norm_quant8(x[:1], w, EPS)
    assert torch.equal(q.a8[-9:], last.a8) and torch.equal(q.s8[:, -9:], last.s8)
    assert (q.a8[:-9] == first.a8).all() and (q.s8[:, :-9] == first.s8).all()


@pytest.mark.parametrize("m", [1, 40, 300, 2049])
def test_bytes_behind_a_rows_last_scale_do_not_count(m):
    g = gen("behind", m)
    (x, _), (w, _) = random_a8(g, m, 1184), random_w8(g, 1056, 1184)
    y = linear_a8(x, w)
    s = x.s8.clone()
    s[-1, :, 1:] = 255  # K = 9 * 128 + 32
    assert torch.equal(linear_a8(A8(x.a8, s), w), y)
