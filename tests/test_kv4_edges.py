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
