"""64-bit reference of the 8-bit activation operators (torch on the CPU), written from their definitions."""
import math

import torch

PERM = [0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15]


def e4m3_values():
    t = []
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = math.nan if b & 127 == 127 else (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
        t.append(-v if b & 128 else v)
    return torch.tensor(t, dtype=torch.float64)


def permuted(codes):
    r, k = codes.shape
    return codes.view(r, k // 16, 16)[:, :, PERM].reshape(r, k).contiguous()


def natural(codes):
    r, k = codes.shape
    inv = [PERM.index(i) for i in range(16)]
    return codes.view(r, k // 16, 16)[:, :, inv].reshape(r, k).contiguous()


def pack_scales(s):
    """[rows, K / 32] bytes -> [ceil(K / 128), rows, 4], 127 behind the last."""
    rows, nb = s.shape
    out = torch.full((rows, -(-nb // 4) * 4), 127, dtype=torch.uint8)
    out[:, :nb] = s
    return out.view(rows, -1, 4).permute(1, 0, 2).contiguous()


def unpack_scales(s, k):
    return s.permute(1, 0, 2).reshape(s.shape[1], -1)[:, :k // 32]


def scale_values(s):
    v = 2.0 ** (s.double() - 127)
    return v.masked_fill(s == 255, math.nan)


def a8_values(a8, s8):
    """Codes [rows, K] in the byte order and packed scales -> float64 values."""
    k = a8.shape[1]
    return e4m3_values()[natural(a8).long()] * scale_values(unpack_scales(s8, k)).repeat_interleave(32, 1)


def w8_values(codes, s8):
    """Codes [N, K] in natural order, scales [ceil(N / 32), K / 32] -> float64 values."""
    n = codes.shape[0]
    return e4m3_values()[codes.long()] * scale_values(s8).repeat_interleave(32, 0)[:n].repeat_interleave(32, 1)


def block_exponents(y):
    """Exponent of each block of 32 of y (float64 [rows, K], finite)."""
    a = y.view(y.shape[0], -1, 32).abs().amax(-1).clamp_min(float(torch.tensor(1e-4, dtype=torch.float32)))
    return torch.ceil(torch.log2(a / 448))


def half_steps(z):
    """Half a step of e4m3 at z (|z| <= 448)."""
    return 2.0 ** (torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 4)


def quantised(y):
    """float64 [rows, K] -> (codes in natural order, E8M0 bytes [rows, K / 32]) of finite y, ties to even."""
    e = block_exponents(y)
    z = (y.view(y.shape[0], -1, 32) / 2.0 ** e.unsqueeze(-1)).reshape(y.shape)
    h = half_steps(z)
    v = torch.round(z / (2 * h)) * 2 * h
    grid = e4m3_values()[:127]
    codes = torch.searchsorted(grid, v.abs().contiguous())
    codes = codes + 128 * torch.signbit(y)
    return codes.to(torch.uint8), (e + 127).to(torch.uint8)


def act(v, name):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "silu":
        return v * torch.special.expit(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))  # (1 + erf would lose the left tail)
    if name == "gelu_tanh":
        return v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))  # (1 + tanh would, too)
    return v


def normed(h, w, eps):
    return h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
