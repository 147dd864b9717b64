"""The 8-bit activation operators of dsv41_amd as cases that can be timed and compared: the norm with the residual's
addition and an 8-bit output (norm_quant8), the block-scaled fp8 product with bias, activation and residual in its
epilogue (linear_a8), the gated product of a feed-forward (gated_a8), and the three as one feed-forward block.

Activations in 8 bits are e4m3 codes with an E8M0 scale per 32 values of a row, weights e4m3 codes with an E8M0 scale
per [32 x 32] block; both hold every 16 values of a row in the byte order ORDER.  An activation's scales are laid out
[ceil(K / 128), rows, 4].  Widths are the attention layer's (5120 wide, its output projection's 8192, its query
latent's 1280 and 32768 columns, 2048), and odd ones between."""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.abspath("deepseekv4.1-a100-custom_amd"))

own = False

DEV = "cuda:0"
BF = torch.bfloat16
EPS = 1e-6
ORDER = [0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15]  # position p of 16 bytes holds value ORDER[p]
BACK = [ORDER.index(i) for i in range(16)]


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's residual stream on its way into a block: latency
        dict(name="norm_1", op="norm", m=1, d=5120, residual=True),
        # the query latent of an odd chunk: short rows, no residual
        dict(name="norm_777_latent", op="norm", m=777, d=1280, residual=False),
        # a long prefill chunk
        dict(name="norm_8192", op="norm", m=8192, d=5120, residual=True),
        # one token's output projection with the residual: a stream of the weights
        dict(name="linear_1", op="linear", m=1, n=5120, k=8192, act="none", bias=False, residual=True, out="bf16"),
        # a serving batch through the query projection
        dict(name="linear_24", op="linear", m=24, n=32768, k=1280, act="none", bias=False, residual=False, out="bf16"),
        # a small odd head: bias and activation, nothing a multiple of a tile
        dict(name="linear_301_odd", op="linear", m=301, n=1001, k=5120 - 96, act="gelu", bias=True, residual=False,
             out="bf16"),
        # a prefill chunk's output projection with the residual
        dict(name="linear_4096", op="linear", m=4096, n=5120, k=8192, act="none", bias=False, residual=True, out="bf16"),
        # one token through the gate and up projections
        dict(name="gated_1", op="gated", m=1, n=8192, k=5120, act="silu", limit=0.0, out="a8"),
        # a batch of users with their drafts, the narrow feed-forward
        dict(name="gated_130", op="gated", m=130, n=2048, k=5120, act="silu", limit=10.0, out="a8"),
        # a prefill chunk
        dict(name="gated_4096", op="gated", m=4096, n=8192, k=5120, act="silu", limit=0.0, out="a8"),
        # the whole block: four users' decode step, and a ragged chunk
        dict(name="ffn_4", op="ffn", m=4, n=8192, k=5120, limit=0.0),
        dict(name="ffn_1999", op="ffn", m=1999, n=8192, k=5120, limit=10.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "gated", "gated", "ffn"])
    if op == "norm":
        return dict(op=op, m=_log(rng, 1, 8192), d=32 * _log(rng, 4, 160), residual=rng.random() < 0.6)
    m, k = _log(rng, 1, 4096), 32 * _log(rng, 16, 256)
    if op == "linear":
        out = rng.choice(["bf16", "bf16", "bf16", "a8"])
        n = _log(rng, 100, min(32768, 8192 * 5120 // k))
        if out == "a8" or rng.random() < 0.5:
            n = 32 * max(1, n // 32)
        return dict(op=op, m=m, n=n, k=k, act=rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.4, residual=out != "a8" and rng.random() < 0.5, out=out)
    n = 32 * _log(rng, 8, min(512, 8192 * 5120 // k // 32))
    if op == "gated":
        return dict(op=op, m=m, n=n, k=k, act=rng.choice(["silu", "silu", "gelu_tanh", "gelu"]),
                    limit=rng.choice([0.0, 7.0, 10.0]), out=rng.choice(["a8", "a8", "bf16"]))
    return dict(op=op, m=min(m, 2048), n=min(n, 8192), k=min(k, 5120), limit=rng.choice([0.0, 10.0]))


# ------------------------------------------------------------------------------------------------ inputs
def _stream(g, m, d):
    """Rows of a residual stream: a few channels are far larger than the others."""
    x = torch.randn(m, d, generator=g, device=DEV)
    x[:, torch.randint(0, d, (max(1, d // 512),), generator=g, device=DEV)] *= 20
    return x


def _weight(g, n, k):
    """An FP8 block-scaled weight as a checkpoint's loader leaves it: codes [n, k] in ORDER, scales [ceil(n/32), k/32]."""
    nb = -(-n // 32)
    w = torch.randn(nb * 32, k, generator=g, device=DEV) * k ** -0.5
    amax = w.view(nb, 32, k // 32, 32).abs().amax((1, 3))
    e = torch.ceil(torch.log2(amax.double() / 448)).to(torch.int32)
    s = torch.exp2(e.float()).repeat_interleave(32, 0).repeat_interleave(32, 1)
    w8 = (w / s).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)[:n]
    return w8.view(n, k // 16, 16)[:, :, ORDER].reshape(n, k).contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29)
    op, m = case["op"], case["m"]
    s = dict(case=case)
    if op in ("norm", "ffn"):
        d = case["d"] if op == "norm" else case["k"]
        s["x"] = _stream(g, m, d).to(BF)
        s["norm"] = (torch.rand(d, generator=g, device=DEV) + 0.5).to(BF)
        if op == "ffn" or case["residual"]:
            s["residual"] = (_stream(g, m, d) * 4).to(BF)
    else:
        s["a8"], s["s8"] = _quant(_stream(g, m, case["k"]))
        s["a8"], s["s8"] = s["a8"].view(torch.uint8), s["s8"].view(torch.uint8)
    if op == "linear":
        s["w"] = _weight(g, case["n"], case["k"])
        s["bias"] = torch.randn(case["n"], generator=g, device=DEV).to(BF) if case["bias"] else None
        s["residual"] = torch.randn(m, case["n"], generator=g, device=DEV).to(BF) if case["residual"] else None
    if op in ("gated", "ffn"):
        s["gate"], s["up"] = _weight(g, case["n"], case["k"]), _weight(g, case["n"], case["k"])
    if op == "ffn":
        s["down"] = _weight(g, case["k"], case["n"])
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _decoded(codes, scale):
    """e4m3 codes in ORDER with the scale of each value -> fp32 values in their own order."""
    r, k = codes.shape
    v = codes.view(torch.float8_e4m3fn).float().view(r, k // 16, 16)[:, :, BACK].reshape(r, k)
    return v * scale


def _activation(a8, s8):
    m, k = a8.shape
    e = s8.permute(1, 0, 2).reshape(m, -1)[:, :k // 32]
    return _decoded(a8, torch.exp2(e.float() - 127).repeat_interleave(32, 1))


def _matrix(w):
    w8, s8 = w
    return _decoded(w8, torch.exp2(s8.float() - 127).repeat_interleave(32, 0)[:w8.shape[0]].repeat_interleave(32, 1))


def _quant(y):
    """fp32 rows -> (codes in ORDER, scales [ceil(K/128), rows, 4]): s = 2^ceil(log2(max(amax, 1e-4) / 448)) per 32."""
    m, k = y.shape
    b = y.view(m, k // 32, 32)
    t = b.abs().amax(-1, keepdim=True).clamp_min(1e-4) / 448
    f, e = torch.frexp(t)
    e = e - (f == 0.5).to(e.dtype)
    codes = torch.ldexp(b, -e).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = codes.view(m, k // 16, 16)[:, :, ORDER].reshape(m, k).view(torch.float8_e4m3fn)
    s = torch.full((m, -(-k // 128) * 4), 127, dtype=torch.uint8, device=y.device)
    s[:, :k // 32] = (e.view(m, k // 32) + 127).to(torch.uint8)
    return codes, s.view(m, -1, 4).permute(1, 0, 2).contiguous().view(torch.float8_e8m0fnu)


def _act(v, act):
    if act == "relu":
        return v * (v > 0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    return v


def _norm(x, residual, w):
    h = x if residual is None else (x.float() + residual.float()).to(BF)
    hf = h.float()
    return h, hf / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS) * w.float()


def _gated(x, gate, up, act, limit):
    g, u = x @ _matrix(gate).t(), x @ _matrix(up).t()
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return _act(g, act) * u


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        h, y = _norm(s["x"], s.get("residual"), s["norm"])
        codes, scales = _quant(y)
        return dict(codes=codes, scales=scales, **(dict(h=h) if c["residual"] else {}))
    if c["op"] == "linear":
        y = _activation(s["a8"], s["s8"]) @ _matrix(s["w"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        y = _act(y, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return dict(zip(("codes", "scales"), _quant(y))) if c["out"] == "a8" else dict(y=y.to(BF))
    if c["op"] == "gated":
        y = _gated(_activation(s["a8"], s["s8"]), s["gate"], s["up"], c["act"], c["limit"])
        return dict(zip(("codes", "scales"), _quant(y))) if c["out"] == "a8" else dict(y=y.to(BF))
    h, y = _norm(s["x"], s["residual"], s["norm"])
    a8, s8 = (t.view(torch.uint8) for t in _quant(y))
    a8, s8 = (t.view(torch.uint8) for t in _quant(_gated(_activation(a8, s8), s["gate"], s["up"], "silu", c["limit"])))
    return dict(y=(_activation(a8, s8) @ _matrix(s["down"]).t() + h.float()).to(BF))


# ------------------------------------------------------------------------------------------------ a pass
def _parts(q):
    return dict(codes=q.a8.view(torch.float8_e4m3fn), scales=q.s8.view(torch.float8_e8m0fnu))


def run(s):
    if not own:
        return _plain(s)
    from dsv41_amd.a8 import A8, gated_a8, linear_a8, norm_quant8
    from dsv41_amd.ffn import GatedFeedForward
    from dsv41_amd.w8 import W8
    c = s["case"]
    if c["op"] == "norm":
        if not c["residual"]:
            return _parts(norm_quant8(s["x"], s["norm"], EPS))
        q, h = norm_quant8(s["x"], s["norm"], EPS, residual=s["residual"])
        return dict(_parts(q), h=h)
    if c["op"] == "linear":
        y = linear_a8(A8(s["a8"], s["s8"]), W8(*s["w"], permuted=True), bias=s["bias"], act=c["act"],
                      residual=s["residual"], out=A8 if c["out"] == "a8" else BF)
        return _parts(y) if c["out"] == "a8" else dict(y=y)
    if c["op"] == "gated":
        y = gated_a8(A8(s["a8"], s["s8"]), W8(*s["gate"], permuted=True), W8(*s["up"], permuted=True), act=c["act"],
                     limit=c["limit"], out=A8 if c["out"] == "a8" else BF)
        return _parts(y) if c["out"] == "a8" else dict(y=y)
    ffn = GatedFeedForward(s["norm"], *(W8(*s[n], permuted=True) for n in ("gate", "up", "down")), eps=EPS,
                           limit=c["limit"])
    return dict(y=ffn(s["x"], residual=s["residual"]))


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, m = case["op"], case["m"]
    a8 = lambda rows, k: rows * k * 33 / 32  # noqa: E731
    w8 = lambda n, k: n * k * 1025 / 1024  # noqa: E731
    if op == "norm":
        d = case["d"]
        return dict(bytes=m * d * (6 if case["residual"] else 2) + a8(m, d) + 2 * d, flops=6 * m * d)
    n, k = case["n"], case["k"]
    if op == "linear":
        size = 33 / 32 if case["out"] == "a8" else 2
        by = a8(m, k) + w8(n, k) + m * n * (size + 2 * case["residual"]) + 2 * n * case["bias"]
        return dict(bytes=by, flops=2 * m * n * k)
    if op == "gated":
        return dict(bytes=a8(m, k) + 2 * w8(n, k) + m * n * (33 / 32 if case["out"] == "a8" else 2), flops=4 * m * n * k)
    return dict(bytes=3 * w8(n, k) + 6 * m * k + 2 * k, flops=6 * m * n * k)


# ------------------------------------------------------------------------------------------------ 64 bits
def _e4m3_table():
    """The value of each of the 256 codes: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f and 0xff are NaN."""
    t = []
    for b in range(256):
        e, f = b >> 3 & 15, b & 7
        v = math.nan if b & 127 == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        t.append(-v if b & 128 else v)
    return torch.tensor(t, dtype=torch.float64, device=DEV)


def _in_order64(v):
    """Rows in ORDER -> rows in their own order."""
    r, k = v.shape
    place = torch.tensor(ORDER, device=DEV).repeat(k // 16) + 16 * torch.div(torch.arange(k, device=DEV), 16, rounding_mode="floor")
    return torch.empty_like(v).index_copy_(1, place, v)


def _spread64(scales, k):
    """Scales [ceil(K/128), rows, 4] as one number a value."""
    col = torch.arange(k, device=DEV)
    return scales[col // 128, :, col // 32 % 4].t()


def _act64(a8, s8):
    one = torch.tensor(2.0, dtype=torch.float64, device=DEV)
    return _in_order64(_e4m3_table()[a8.long()]) * _spread64(torch.pow(one, s8.double() - 127), a8.shape[1])


def _weight64(w):
    v = _in_order64(_e4m3_table()[w[0].long()])
    sc = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEV), w[1].double() - 127)
    rows = torch.arange(v.shape[0], device=DEV) // 32
    cols = torch.arange(v.shape[1], device=DEV) // 32
    return v * sc[rows][:, cols]


def _quant64(y):
    """The nearest e4m3 values (ties to the even code) of y over its block's power of two, as 64-bit numbers."""
    m, k = y.shape
    top = y.unflatten(1, (-1, 32)).abs().max(2).values
    top = torch.maximum(top, top.new_tensor(1e-4))
    scales = torch.ones(m, -(-k // 128) * 4, dtype=torch.float64, device=DEV)
    scales[:, :k // 32] = 2.0 ** torch.ceil(torch.log2(top / 448))
    scales = scales.unflatten(1, (-1, 4)).transpose(0, 1).contiguous()
    z = y / _spread64(scales, k)
    step = 2.0 ** (torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
    z = (torch.round(z / step) * step).clamp(-448, 448)
    col = torch.arange(k, device=DEV)
    return z[:, col // 16 * 16 + torch.tensor(ORDER, device=DEV)[col % 16]], scales


def _act_fn64(v, act):
    if act == "none":
        return v
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "silu":
        return v * torch.special.expit(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    return v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))


def _norm64(s, residual):
    h = s["x"].double()
    if residual is not None:
        h = (h + residual.double()).to(BF).double()  # (the stream holds bf16, and the norm is the stream's)
    return h, h * s["norm"].double() / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt()


def _gated64(x, s, act, limit):
    g, u = x @ _weight64(s["gate"]).t(), x @ _weight64(s["up"]).t()
    if limit:
        g, u = torch.minimum(g, g.new_tensor(limit)), torch.maximum(torch.minimum(u, u.new_tensor(limit)), u.new_tensor(-limit))
    return _act_fn64(g, act) * u


def _codes64(codes, scales):
    """The values that codes in ORDER and their scales stand for."""
    return _in_order64(codes) * _spread64(scales, codes.shape[1])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h, y = _norm64(s, s.get("residual"))
        codes, scales = _quant64(y)
        return dict(codes=codes, scales=scales, **(dict(h=s["x"].double() + s["residual"].double()) if case["residual"] else {}))
    if op == "linear":
        y = _act64(s["a8"], s["s8"]) @ _weight64(s["w"]).t()
        if case["bias"]:
            y = y + s["bias"].double()
        y = _act_fn64(y, case["act"])
        if case["residual"]:
            y = y + s["residual"].double()
        return dict(zip(("codes", "scales"), _quant64(y))) if case["out"] == "a8" else dict(y=y)
    if op == "gated":
        y = _gated64(_act64(s["a8"], s["s8"]), s, case["act"], case["limit"])
        return dict(zip(("codes", "scales"), _quant64(y))) if case["out"] == "a8" else dict(y=y)
    h, y = _norm64(s, s["residual"])
    a = _codes64(*_quant64(y))
    a = _codes64(*_quant64(_gated64(a, s, "silu", case["limit"])))
    return dict(y=h + a @ _weight64(s["down"]).t())
