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


# (rows, heads, list, window, rows of the cache's tables) of prompts whose cache is decoded first, and of some just short of it
FIRST = [(530, 33, 256, 100, 256), (530, 64, 256, 1, 256), (530, 80, 250, 37, 256), (531, 64, 257, 128, 2016), (130, 64, 1025, 128, 2304),
         (68, 128, 2000, 64, 2176), (520, 40, 260, 0, 416)]
DIRECT = [(530, 32, 256, 100, 256), (150, 33, 512, 128, 650), (15, 64, 9000, 128, 416), (530, 64, 256, 100, 40000), (65529, 64, 256, 1, 256)]


@pytest.mark.parametrize("first,args", [(True, a) for a in FIRST] + [(False, a) for a in DIRECT])
def test_which_prompts_are_decoded_first(first, args):
    """More than 32 heads, 16 to 65528 query rows, 2^18 keys of 16 heads, and each row of the cache's tables listed four times: the
    workspace then holds the tables' rows in bf16 (else the splits' partial results, of few rows)."""
    rows, heads, t, w, held = args
    c = ctypes.byref(_struct(dim=576, page=16, pages=4096, slots=1, cols=held // 16))
    n = _lib.lib().dsv41_kv4_attn_workspace_bytes(c, rows, heads, w, t, 1)
    decoded = held // 16 * 16 * 576 * 2
    assert n >= decoded + rows * (w + t) * 4 if first else n % (4 * rows * heads * 514) == 0
