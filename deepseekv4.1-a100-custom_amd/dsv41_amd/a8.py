"""Activations in 8 bits and the operators on them: the twin of the W8 weights (dsv41/w8.py:39-60) for x.

fake_quant_fp8 / norm_quant put activations ON the fp8 grid and keep them in bf16; here they are held as the grid's own
bytes -- e4m3 codes with one E8M0 scale per 32 values of a row -- which the products turn into bf16 in registers, exactly,
beside the weights.  What stands between the attention layer and the next one is then three launches:

  q, h = norm_quant8(x, w, eps, residual=r)     h = x + r, q = rmsnorm(h) * w in 8 bits
  a    = gated_a8(q, w_gate, w_up)              silu(q Wg^T) * (q Wu^T) in 8 bits
  y    = linear_a8(a, w_down, residual=h)       a Wd^T + h

Forward only, as everything here: inputs that require a gradient are refused while gradients are recorded."""
from __future__ import annotations

import math

import torch

from ._lib import as_bf16, call, ptr, require_gpu, stream_of
from .w8 import W8, unpermute_k

MOST = 0x7fffff00  # rows and columns of a product
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


class A8:
    """8-bit activations of `shape` [..., K], K % 32 == 0: a8 uint8 [rows, K], e4m3 bits with every 16 of a row in the
    weights' byte order (w8.PERM_K); s8 uint8 [ceil(K / 128), rows, 4], E8M0 (2^(byte - 127)): byte j of word (c, row) is
    the scale of values 128 c + 32 j .. + 31 of that row, 127 where K ends before them.  A block that held an infinity or
    a NaN has scale 255 and NaN codes."""
    __slots__ = ("a8", "s8", "shape")

    def __init__(self, a8: torch.Tensor, s8: torch.Tensor, shape: tuple | None = None):
        if a8.dtype != torch.uint8 or s8.dtype != torch.uint8 or a8.dim() != 2 or a8.shape[1] % 32:
            raise ValueError("A8: uint8 codes [rows, K] with K % 32 == 0 and uint8 scales expected")
        rows, k = a8.shape
        if s8.shape != ((k + 127) // 128, rows, 4):
            raise ValueError(f"A8: scales {tuple(s8.shape)} for codes {tuple(a8.shape)}: [ceil(K / 128), rows, 4] expected")
        if s8.device != a8.device:
            raise RuntimeError(f"A8: codes on {a8.device}, scales on {s8.device}")
        if shape is not None and (len(shape) == 0 or shape[-1] != k or math.prod(shape[:-1]) != rows):
            raise ValueError(f"A8: shape {tuple(shape)} for codes {tuple(a8.shape)}")
        self.a8, self.s8 = a8.contiguous(), s8.contiguous()
        self.shape = tuple(a8.shape) if shape is None else tuple(shape)

    @property
    def device(self):
        return self.a8.device

    def scales(self) -> torch.Tensor:
        """E8M0 bytes [rows, K / 32] of the blocks in order."""
        rows, k = self.a8.shape
        return self.s8.permute(1, 0, 2).reshape(rows, -1)[:, :k // 32]

    def float(self) -> torch.Tensor:
        """The values, fp32 [..., K] (exact)."""
        rows, k = self.a8.shape
        e = self.scales().to(torch.int32)
        s = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127).masked_fill_(e == 255, float("nan"))
        v = unpermute_k(self.a8).view(torch.float8_e4m3fn).float().view(rows, k // 32, 32) * s.unsqueeze(-1)
        return v.view(self.shape)

    def bf16(self) -> torch.Tensor:
        """The values as bf16 [..., K] (exact, as fake_quant_fp8's): x of fp8_gemm_tc."""
        return self.float().to(torch.bfloat16)


def _index(*ts: torch.Tensor | None) -> int:
    """The index of the GPU that the tensors are on (the first is one); raises as require_gpu does."""
    i = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != i:
            require_gpu(*ts)
    if i < 0:
        require_gpu(*ts)
    return i


def _no_grad(name: str, *ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name}: forward only (an input requires a gradient)")


def _aligned(t: torch.Tensor, n: int = 16) -> torch.Tensor:
    return t if t.data_ptr() % n == 0 else t.clone()


def _codes(rows: int, k: int, dev: torch.device, shape: tuple) -> A8:
    q = A8.__new__(A8)
    q.a8 = torch.empty(rows, k, dtype=torch.uint8, device=dev)
    q.s8 = torch.empty((k + 127) // 128, rows, 4, dtype=torch.uint8, device=dev)
    q.shape = shape
    return q


def _launch(name: str, index: int, *args) -> None:
    """The call on the current stream of GPU `index`, with that GPU current."""
    if index == torch.cuda.current_device():
        call(name, *args, stream_of(index))
    else:
        with torch.cuda.device(index):
            call(name, *args, stream_of(index))


def norm_quant8(x: torch.Tensor, w: torch.Tensor | None, eps: float, residual: torch.Tensor | None = None):
    """rmsnorm(x + residual) * w in 8 bits, the residual's addition and the norm (dsv41/fused2.py:251-272) in one pass.

    x, residual: bf16 [..., D], D % 32 == 0, D <= 16384; w: [D], rounded to bf16 where it is not (as rmsnorm and
    norm_quant do), or None (no norm: the quantisation alone).  Returns the A8, with a residual (A8, h): h = bf16(x +
    residual), the stream that the norm is of.  The normed value is rounded once, to 8 bits (norm_quant rounds to bf16 in
    between, as the reference does, so single codes differ from its)."""
    index = _index(x, residual, w)
    _no_grad("norm_quant8", x, residual, w)
    shape = x.shape
    D = shape[-1] if shape else 0
    if x.dtype != torch.bfloat16 or (residual is not None and residual.dtype != torch.bfloat16):
        raise RuntimeError("norm_quant8: bf16 rows expected")
    if D == 0 or D % 32 or D > 16384:
        raise RuntimeError(f"norm_quant8: rows of {D} (a multiple of 32, at most 16384)")
    if residual is not None and residual.shape != shape:
        raise RuntimeError(f"norm_quant8: residual {tuple(residual.shape)} for x {tuple(shape)}")
    if w is not None:
        if w.dim() != 1 or w.shape[0] != D:
            raise RuntimeError(f"norm_quant8: weight {tuple(w.shape)} for rows of {D}")
        w = _aligned(as_bf16(w))
    x = _aligned(x.contiguous())
    rows = x.numel() // D
    q = _codes(rows, D, x.device, shape)
    if residual is None:
        _launch("dsv41_norm_quant8", index, x.data_ptr(), None, ptr(w), eps, None, q.a8.data_ptr(), q.s8.data_ptr(), rows, D)
        return q
    residual = _aligned(residual.contiguous())
    h = torch.empty_like(x)
    _launch("dsv41_norm_quant8", index, x.data_ptr(), residual.data_ptr(), ptr(w), eps, h.data_ptr(), q.a8.data_ptr(),
            q.s8.data_ptr(), rows, D)
    return q, h


def _operands(name: str, x: A8, act: str, out, w: W8):
    """Checks of one weight; its columns and K."""
    if not isinstance(x, A8) or not isinstance(w, W8):
        raise TypeError(f"{name}: an A8 and W8 weights expected")
    if act not in ACTS:
        raise ValueError(f"{name}: act {act!r} (one of {', '.join(ACTS)})")
    if out is not A8 and out is not torch.bfloat16:
        raise ValueError(f"{name}: out {out} (torch.bfloat16 or A8; fp32 sums: w8.fp8_gemm_tc)")
    K = x.shape[-1]
    N, Kw = w.shape
    s = w.s8.shape
    if Kw != K or K > 32768 or len(s) != 2 or s[0] < (N + 31) // 32 or s[1] < K // 32:
        raise RuntimeError(f"{name}: weight {(N, Kw)}, scales {tuple(s)} for x {tuple(x.shape)} (K at most 32768)")
    if N > MOST or x.a8.shape[0] > MOST:
        raise RuntimeError(f"{name}: {x.a8.shape[0]} rows, {N} columns (at most {MOST})")
    if out is A8 and N % 32:
        raise RuntimeError(f"{name}: {N} columns in 8 bits (a multiple of 32)")
    return N, K


def _output(x: A8, N: int, out, dev: torch.device):
    """The result, and its three pointers."""
    shape = (*x.shape[:-1], N)
    if out is A8:
        y = _codes(x.a8.shape[0], N, dev, shape)
        return y, None, y.a8.data_ptr(), y.s8.data_ptr()
    y = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    return y, y.data_ptr(), None, None


def linear_a8(x: A8, w: W8, bias: torch.Tensor | None = None, act: str = "none", residual: torch.Tensor | None = None,
              out=torch.bfloat16):
    """act(x W^T + bias) + residual -> [..., N] bf16, or (out=A8) in 8 bits.

    x: A8 [..., K]; w: W8 [N, K]; bias: [N] bf16 or fp32; act: none, relu, silu, gelu (erf), gelu_tanh; residual: bf16
    [..., N].  fp32 sums; bias, activation and residual are applied to them and the result is rounded once."""
    N, K = _operands("linear_a8", x, act, out, w)
    xa, xs, wa, ws = x.a8, x.s8, w.w8, w.s8
    index = _index(xa, xs, wa, ws, bias, residual)
    bias_f32 = 0
    if bias is not None:
        if bias.shape != (N,) or bias.dtype not in (torch.bfloat16, torch.float32):
            raise RuntimeError(f"linear_a8: bias {tuple(bias.shape)} {bias.dtype} (bf16 or fp32 [{N}])")
        _no_grad("linear_a8", bias)
        bias_f32 = int(bias.dtype == torch.float32)
        bias = bias.contiguous()
    if residual is not None:
        if residual.shape != (*x.shape[:-1], N) or residual.dtype != torch.bfloat16:
            raise RuntimeError(f"linear_a8: residual {tuple(residual.shape)} {residual.dtype} (bf16 {(*x.shape[:-1], N)})")
        _no_grad("linear_a8", residual)
        residual = residual.contiguous()
    if (xa.data_ptr() | wa.data_ptr()) & 15 or xs.data_ptr() & 3:
        xa, xs, wa = _aligned(xa), _aligned(xs, 4), _aligned(wa)
    y, o, oa, os = _output(x, N, out, xa.device)
    _launch("dsv41_linear_a8", index, xa.data_ptr(), xs.data_ptr(), wa.data_ptr(), ws.data_ptr(), xa.shape[0], N, K,
            ws.shape[1], ptr(bias), bias_f32, ACTS[act], ptr(residual), o, oa, os)
    return y


def gated_a8(x: A8, w_gate: W8, w_up: W8, act: str = "silu", limit: float = 0.0, out=A8):
    """The gated product of a feed-forward, act(x Wg^T) * (x Wu^T) -> [..., N] in 8 bits, or (out=torch.bfloat16) bf16.

    x: A8 [..., K]; w_gate, w_up: W8 [N, K]; act as linear_a8's.  limit > 0: the gate's sum is held to at most limit and
    the up sum to [-limit, limit] first.  Both sums stay in registers; the result is rounded once."""
    N, K = _operands("gated_a8", x, act, out, w_gate)
    if _operands("gated_a8", x, act, out, w_up) != (N, K):
        raise RuntimeError(f"gated_a8: gate {w_gate.shape}, up {w_up.shape}")
    if not limit >= 0.0:
        raise ValueError(f"gated_a8: limit {limit} (0: none)")
    if limit > 0.0:
        limit = max(limit, 2.0 ** -149)  # (fp32's smallest number: less would be 0, no limit)
    xa, xs, ga, gs, ua, us = x.a8, x.s8, w_gate.w8, w_gate.s8, w_up.w8, w_up.s8
    index = _index(xa, xs, ga, gs, ua, us)
    if (xa.data_ptr() | ga.data_ptr() | ua.data_ptr()) & 15 or xs.data_ptr() & 3:
        xa, xs, ga, ua = _aligned(xa), _aligned(xs, 4), _aligned(ga), _aligned(ua)
    y, o, oa, os = _output(x, N, out, xa.device)
    _launch("dsv41_gated_a8", index, xa.data_ptr(), xs.data_ptr(), ga.data_ptr(), gs.data_ptr(), ua.data_ptr(),
            us.data_ptr(), xa.shape[0], N, K, gs.shape[1], us.shape[1], ACTS[act], limit, o, oa, os)
    return y
