"""The paged 4-bit cache on the CPU: index lists of every integer type, launch limits, which kernel takes a prompt."""
import ctypes

import pytest
import torch

from dsv41_amd import _lib, kv4
from test_kv4 import _cache, _struct

BF = torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8])
def test_index_lists_of_every_integer_type(dtype):
    want = [[[5, 0, 100, 255]]] if dtype == torch.uint8 else [[[5, -1, 100, 127]]]
    got, t = kv4._indices("x", torch.tensor(want, dtype=dtype), (1, 1), -1)
    assert t == 4 and got.dtype == torch.int32 and got.tolist() == want


def test_window_of_one_batch_row():
    """A batch of one has any batch stride; the entry points take multiples of 8."""
    odd = torch.zeros(5 * 576 + 4, dtype=BF).as_strided((1, 5, 576), (5 * 576 + 4, 576, 1))
    assert odd.stride(0) % 8 and kv4._window("x", odd, 576).stride(0) % 8 == 0
    assert kv4._window("x", torch.zeros(3, 0, 576, dtype=BF), 576).shape == (3, 0, 576)


def test_launches_of_too_many_lanes_are_refused():
    """2^32 lanes and more in one launch are turned away with the arguments, not by the runtime."""
    L, P, inv = _lib.lib(), 1 << 20, 1
    c = ctypes.byref(_struct())
    assert L.dsv41_kv4_append(c, P, 512, P, P, 1 << 27, 4, 0, P, P, 9, 64, None) == inv
    assert L.dsv41_kv4_read(c, P, P, 1 << 27, P, None) == inv
    assert L.dsv41_kv4_fork(c, P, P, None, 1 << 24, None) == inv
    assert L.dsv41_kv4_release(c, P, None, 1 << 24, None) == inv
    assert L.dsv41_kv4_copy(c, ctypes.byref(_struct(pool=1 << 40)), P, P, 1 << 24, P, 1 << 40, None) == inv
    assert L.dsv41_sattn4(c, P, P, 128 * 512, 2, 128, P, 10, P, P, P, None, P, P, P, 100, 64, 1.0, P, 1 << 24, 1, None, 0, None) == inv
    assert L.dsv41_sparse_attn4(c, P, P, 128 * 512, 128, P, 0, P, 10, None, P, 1.0, P, 1, 1 << 24, 1, None, 0, None) == inv
    one, h = torch.zeros(1, dtype=torch.int64), _cache()
    for n in (1 << 24, 1 << 32):
        many = one.expand(n)
        for call in (lambda: h.fork(many, many), lambda: h.release(many), lambda: h.copy_pages(other, many, many)):
            other = _cache()
            h._span, other._span = (0, 10), (10, 20)
            with pytest.raises(RuntimeError, match="at most"):
                call()
