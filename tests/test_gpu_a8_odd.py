"""Gated products whose columns end inside a 32-column block (bf16 output) on every kernel that takes more than 32 rows:
the last block's gate, up and scale rows are held inside the weights, columns past the end are not stored."""
import pytest

import _a8_ref as R
from dsv41_amd import gated_a8
from dsv41_amd.w8 import W8
from test_gpu_a8 import ACT_ERR, BF, DEV, check_bf16, gen, whole_a8, whole_w8
from test_gpu_a8_sums import check_plan

pytestmark = pytest.mark.gpu

# 8 n columns behind the last block, or an odd number
SIZES = [(129, 417, 5120, (0, 32, 64, False)), (140, 1940, 160, (0, 48, 64, False)), (200, 2008, 352, (0, 64, 64, False)),
         (2049, 281, 224, (1, 128, 64, False)), (2049, 264, 224, (1, 128, 64, False)), (1100, 1049, 160, (1, 128, 128, False)),
         (1100, 1032, 160, (1, 128, 128, False)), (1024, 4045, 640, (1, 256, 128, False)), (1024, 4040, 640, (1, 256, 128, False)),
         (2049, 2037, 1312, (1, 192, 256, False)), (2049, 2024, 1312, (1, 192, 256, False)), (4090, 2011, 1280, (1, 256, 256, False)),
         (4090, 2000, 1280, (1, 256, 256, False)), (4090, 2523, 160, (1, 256, 256, True)), (4090, 2504, 160, (1, 256, 256, True))]


@pytest.mark.parametrize("m,n,k,kind", SIZES)
def test_gated_columns_that_end_inside_a_block(m, n, k, kind):
    check_plan(m, n, k, kind, gated=True)
    g = gen("gated odd", m, n, k)
    (x, xv), (wg, gv), (wu, uv) = whole_a8(g, m, k), whole_w8(g, n, k), whole_w8(g, n, k)
    wg, wu = W8(wg.w8, wg.s8 - 6, permuted=True), W8(wu.w8, wu.s8 - 4, permuted=True)
    gate, up = ((xv.to(DEV) @ v.to(DEV).t()).cpu() / d for v, d in ((gv, 64), (uv, 16)))
    want = R.act(gate, "silu") * up
    check_bf16(gated_a8(x, wg, wu, out=BF), want, want.abs() * (ACT_ERR + 2.0 ** -23) + 1e-30)
    want = R.act(gate.clamp(max=0.5), "gelu") * up.clamp(-0.5, 0.5)
    y = gated_a8(x, wg, wu, act="gelu", limit=0.5, out=BF)
    assert y.shape == (m, n) and y.is_contiguous()
    check_bf16(y, want, want.abs() * (ACT_ERR + 2.0 ** -23) + 1e-30)
