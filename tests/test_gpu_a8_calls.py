"""Calls of the 8-bit activation operators at the ends of what their arguments allow."""
import pytest

from dsv41_amd import gated_a8
from test_gpu_a8 import BF, gen, whole_a8, whole_w8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 20, 40, 300])
@pytest.mark.parametrize("limit", [1e-40, 1e-45, 1e-46, 1e-300])
def test_a_limit_below_fp32_is_a_limit(m, limit):
    """Sums are below 2^16 (128 products of at most 16) and |up| is held to 1e-40 < 2^-132 or less."""
    g = gen("limit", m)
    (x, _), (wg, _), (wu, _) = whole_a8(g, m, 128), whole_w8(g, 64, 128), whole_w8(g, 64, 128)
    free = gated_a8(x, wg, wu, act="none", out=BF)
    held = gated_a8(x, wg, wu, act="none", limit=limit, out=BF)
    assert free.abs().max() > 1 and held.float().abs().max() <= 2.0 ** -116
