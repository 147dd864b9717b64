"""Bias, activation and residual of linear_a8 against 64 bits on every kernel that takes more than 32 rows, in rows of whole
16-byte units (N % 8 == 0: vector loads and stores) and in others; the residual under an 8-bit output.

Sums are exact (whole numbers), so is the bias's addition but for one rounding to fp32, which the reference makes too; the
activation is off by ACT_ERR relative at most, the residual's addition rounds once (2^-24; 2^-23 is allowed), the output once."""
import pytest
import torch

import _a8_ref as R
from dsv41_amd import A8, linear_a8
from dsv41_amd.w8 import W8
from test_gpu_a8 import ACT_ERR, BF, DEV, bf, check_a8, check_bf16, gen, whole_a8, whole_w8
from test_gpu_a8_sums import check_plan

pytestmark = pytest.mark.gpu

T64, T128, T256, T192x256, T256x256 = [(1, *t, False) for t in ((128, 64), (128, 128), (256, 128), (192, 256), (256, 256))]
SIZES = [(130, 2048, 5120, (0, 48, 32, False), "gelu"), (300, 1280, 288, (0, 64, 32, False), "silu"),
         (257, 260, 352, (0, 48, 32, False), "relu"), (64, 257, 1280, (0, 32, 32, False), "gelu_tanh"),
         (2049, 512, 288, T64, "gelu"), (2049, 513, 288, T64, "silu"), (2100, 1056, 1184, T128, "silu"),
         (2100, 1051, 1184, T128, "none"), (1024, 8160, 640, T256, "gelu_tanh"), (1024, 8157, 640, T256, "relu"),
         (2049, 4096, 1312, T192x256, "relu"), (2049, 4090, 1312, T192x256, "gelu"), (4090, 4064, 1280, T256x256, "silu"),
         (4090, 4060, 1280, T256x256, "gelu_tanh"), (2049, 7232, 160, (*T192x256[:3], True), "gelu"),
         (2049, 7233, 160, (*T192x256[:3], True), "silu"), (4090, 4928, 160, (*T256x256[:3], True), "none")]


@pytest.mark.parametrize("m,n,k,kind,act", SIZES)
def test_linear_epilogue_of_every_kernel(m, n, k, kind, act):
    check_plan(m, n, k, kind)
    g = gen("tile epilogue", m, n, k)
    (x, xv), (w, wv) = whole_a8(g, m, k), whole_w8(g, n, k)
    w = W8(w.w8, w.s8 - 6, permuted=True)  # (sums of a size at which the activations bend)
    pre = (xv.to(DEV) @ wv.to(DEV).t()).cpu() / 64
    r = bf(g, m, n)
    for bias in (None, BF, torch.float32):
        b, p = None, pre
        if bias is not None:
            b = torch.randn(n, generator=g).to(bias)
            p = (pre.float() + b.float()).double()
        y0 = R.act(p, act)
        y1 = y0 + r.double()
        err = y0.abs() * ACT_ERR + y1.abs() * 2.0 ** -23 + 1e-30
        kw = dict(bias=None if b is None else b.to(DEV), act=act, residual=r.to(DEV))
        check_bf16(linear_a8(x, w, **kw), y1, err)
        if n % 32 == 0:
            check_a8(linear_a8(x, w, out=A8, **kw), y1, err)
    check_bf16(linear_a8(x, w, act=act), R.act(pre, act), R.act(pre, act).abs() * ACT_ERR + 1e-30)


@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("n", [64, 96])
def test_residual_under_8_bit_output_of_few_rows(m, n):
    g = gen("a8 residual", m, n)
    (x, xv), (w, wv) = whole_a8(g, m, 416), whole_w8(g, n, 416)
    r = bf(g, m, n, scale=30.0)
    want = xv @ wv.t() + r.double()
    check_a8(linear_a8(x, w, residual=r.to(DEV), out=A8), want, want.abs() * 2.0 ** -23)
