"""The sums of the 8-bit products against 64 bits on every kernel that takes more than 32 rows: as exact as fp32's.

A bf16 output shows 8 bits of a sum.  With -bf16(sum) as the residual it shows what the sum has below them: the residual's
addition is exact (two numbers within a factor of two), what is left is 2^-8 of the sum at most and is rounded by 2^-8 of
that.  In the 2-norm both factors are uniform in their range, 1 / sqrt 3 of its end: 2^-16 / 3 of the sums' norm.  The
sum itself is of exact products in fp32: one rounding by 2^-24 for every 32 k and some for the partial sums' joining, in the
2-norm twice sqrt(K / 32 + 8) 2^-24 at most; a single one within (K / 32 + 32) 2^-23 of the sum of magnitudes."""
import pytest
import torch

import _a8_ref as R
from dsv41_amd import A8, gated_a8, linear_a8
from dsv41_amd.w8 import W8
from test_gpu_a8 import BF, DEV, gen, plan, random_a8, random_w8, whole_a8, whole_w8

pytestmark = pytest.mark.gpu

# (rows, columns, k) and the kernel: tile, rows, weight rows of a workgroup; True: with a second launch
LINEAR = [(127, 128, 2080, (0, 32, 32, False)), (130, 2048, 5120, (0, 48, 32, False)), (300, 1280, 288, (0, 64, 32, False)),
          (64, 8192, 8192, (0, 64, 32, False)), (2049, 512, 288, (1, 128, 64, False)), (2100, 1056, 1184, (1, 128, 128, False)),
          (450, 4640, 6176, (1, 128, 128, False)), (1024, 8160, 640, (1, 256, 128, False)), (2049, 4096, 1312, (1, 192, 256, False)),
          (4090, 4064, 1280, (1, 256, 256, False)), (2049, 7232, 160, (1, 192, 256, True)), (4090, 4928, 160, (1, 256, 256, True))]
GATED = [(129, 416, 5120, (0, 32, 64, False)), (450, 2336, 6176, (0, 48, 64, False)), (200, 2016, 352, (0, 64, 64, False)),
         (2049, 288, 224, (1, 128, 64, False)), (1100, 1056, 160, (1, 128, 128, False)), (1024, 4064, 640, (1, 256, 128, False)),
         (2049, 2048, 1312, (1, 192, 256, False)), (4090, 2016, 1280, (1, 256, 256, False)), (4090, 2528, 160, (1, 256, 256, True))]


def check_plan(m, n, k, kind, gated=False):
    p = plan(m, n, k, gated=gated)
    assert (p >> 30, p >> 16 & 0x3fff, p >> 4 & 0xfff, plan(m, n, k, gated=gated, rest=True) != 0) == kind


def rms(t):
    return t.pow(2).mean().sqrt().item()


@pytest.mark.parametrize("m,n,k,kind", LINEAR)
def test_linear_sums_are_as_exact_as_fp32(m, n, k, kind):
    check_plan(m, n, k, kind)
    g = gen("sums", m, n, k)
    (x, xv), (w, wv) = random_a8(g, m, k), random_w8(g, n, k)
    xv, wv = xv.to(DEV), wv.to(DEV)
    want = xv @ wv.t()
    res = -want.to(BF)
    low = want + res.double()
    y = linear_a8(x, w, residual=res).double()
    off = (y - low).abs()
    mags = xv.abs() @ wv.abs().t()
    assert (off <= low.abs() * 2.0 ** -8 + mags * ((k / 32 + 32) * 2.0 ** -23)).all()
    tol = 1.05 * 2.0 ** -16 / 3 + 2 * (k / 32 + 8) ** 0.5 * 2.0 ** -24
    assert rms(off) <= tol * rms(want), (rms(off) / rms(want), tol)


@pytest.mark.parametrize("m,n,k,kind", LINEAR)
def test_large_products_that_cancel_leave_the_others_exact(m, n, k, kind):
    """Whole numbers times 2^-2 with two products of 802816 (22 bits in all: fp32 holds every partial sum), in the first and
    the last block of k, of opposite sign: the result is the other products', bit for bit."""
    check_plan(m, n, k, kind)
    g = gen("cancel", m, n, k)
    (x, xv), (w, wv) = whole_a8(g, m, k), whole_w8(g, n, k)
    nat, wnat, s, ws = R.natural(x.a8.cpu()), R.natural(w.w8.cpu()), R.unpack_scales(x.s8.cpu(), k).clone(), w.s8.cpu().clone()
    a, b = 5, k - 7
    s[:, 0], s[:, -1], ws[:, 0], ws[:, -1] = 128, 128, 128, 128
    nat[:, a], nat[:, b], wnat[:, a], wnat[:, b] = 0x7e, 0x7e, 0x7e, 0xfe
    x, w = A8(R.permuted(nat).to(DEV), R.pack_scales(s).to(DEV)), W8(wnat.to(DEV), ws.to(DEV))
    xv, wv = R.a8_values(R.permuted(nat), R.pack_scales(s)).to(DEV), R.w8_values(wnat, ws).to(DEV)
    assert (xv[0, a] * wv[0, a]).item() == 802816 and (xv[0, b] * wv[0, b]).item() == -802816
    assert torch.equal(linear_a8(x, w), (xv @ wv.t()).to(BF))


@pytest.mark.parametrize("m,n,k,kind", GATED)
def test_gated_codes_are_those_of_fp32_sums(m, n, k, kind):
    """silu(g) u in 8 bits against the quantised 64-bit product.  A code differs where the product's error reaches over a
    rounding border: with a relative error e and steps of at most 2^-3 of a value, the squares of the differences add up to at
    most 2 e 2^-3 of the values'.  e: two sums of 2 sqrt(K / 32 + 8) 2^-24 (2.4e-6 together at K 6176), silu's 3 |g| + 6
    roundings of 2^-24 (e^-g of a g off by 3 of them; 2.1e-6 at |g| = 10): under 2^-17.5, so 2^-9.75 in the 2-norm."""
    check_plan(m, n, k, kind, gated=True)
    g = gen("gated sums", m, n, k)
    (x, xv), (wg, gv), (wu, uv) = random_a8(g, m, k), random_w8(g, n, k), random_w8(g, n, k)
    xv = xv.to(DEV)
    want = (R.act(xv @ gv.to(DEV).t(), "silu") * (xv @ uv.to(DEV).t())).cpu()
    codes, s = R.quantised(want)
    want = R.a8_values(R.permuted(codes), R.pack_scales(s))
    q = gated_a8(x, wg, wu)
    got = R.a8_values(q.a8.cpu(), q.s8.cpu())
    assert rms(got - want) <= 2.0 ** -9.75 * rms(want), rms(got - want) / rms(want)
