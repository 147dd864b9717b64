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
