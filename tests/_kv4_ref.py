"""The paged 4-bit cache and its attention in 64 bits, from their definitions, on the CPU."""
import numpy as np
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
ROW_BYTES = {512: 288, 576: 336}


def grid(y: torch.Tensor):
    """fp64 rows [n, d] -> (values on the grid, codes [n, d], scale bytes [n, d / 16]); groups that hold an infinity or a
    NaN are NaN."""
    n, d = y.shape
    z = y.double().view(n, d // 16, 16)
    bad = ~torch.isfinite(z).all(-1, keepdim=True)
    z = torch.where(bad, torch.zeros_like(z), z)
    t = (z.abs().amax(-1, keepdim=True).clamp_min(6 / 512) / 6.0).clamp(max=448.0)
    s = t.to(torch.float32).to(torch.float8_e4m3fn)
    w = (z.abs() / s.double()).clamp(max=6.0)
    c = torch.where(w < 2, torch.round(w * 2), torch.where(w < 4, torch.round(w) + 2, torch.round(w / 2) + 4)).long()
    v = torch.tensor(E2M1, dtype=torch.float64)[c] * s.double() * torch.where(z < 0, -1.0, 1.0)
    c = torch.where(bad, torch.zeros_like(c), c + 8 * (z < 0))
    v = torch.where(bad, torch.full_like(v, float("nan")), v)
    s = torch.where(bad[..., 0], torch.full_like(bad[..., 0], 0x7f, dtype=torch.uint8), s[..., 0].view(torch.uint8))
    return v.view(n, d), c.view(n, d).to(torch.uint8), s


def pack(y: torch.Tensor) -> torch.Tensor:
    """Rows [n, 512 or 576] -> packed rows uint8 [n, 288 or 336]."""
    _, c, s = grid(y)
    n, d = y.shape
    two = c[:, 0::2] | c[:, 1::2] << 4
    out = torch.zeros(n, ROW_BYTES[d], dtype=torch.uint8)
    out[:, :256], out[:, 256:288] = two[:, :256], s[:, :32]
    if d == 576:
        out[:, 288:320], out[:, 320:324] = two[:, 256:], s[:, 32:]
    return out


def rotate(x: torch.Tensor, cos, sin, pos, rd: int, inverse: bool = False) -> torch.Tensor:
    """fp64 rows [..., d] at position pos: the last rd columns, pairs (2j, 2j + 1)."""
    if rd == 0:
        return x.clone()
    y = x.clone()
    c, s = cos[pos].double(), sin[pos].double() * (-1 if inverse else 1)
    a, b = x[..., -rd::2], x[..., x.shape[-1] - rd + 1::2]
    y[..., -rd::2], y[..., x.shape[-1] - rd + 1::2] = a * c - b * s, a * s + b * c
    return y


def attend(q, rows, sink, scale):
    """q [h, d], rows [t, d] (those that are there), sink [h], all fp64 -> [h, 512]; zeros without a row."""
    if rows.shape[0] == 0:
        return torch.zeros(q.shape[0], 512, dtype=torch.float64)
    x = torch.cat((q @ rows.t() * scale, sink[:, None]), 1)
    return x.softmax(1)[:, :-1] @ rows[:, :512]


def ring_slots(pos: int, pmax: int, plim: int, W: int):
    """The ring's slots that a query sees: slot j holds the newest position <= pmax that is j modulo W."""
    out = []
    for j in range(W):
        held = pmax - (pmax - j) % W
        if 0 <= held <= plim and pos - held < W:
            out.append(j)
    return out


class Model:
    """A cache as Python lists: every sequence's pages, every page's users."""

    def __init__(self, pages, slots, cols, page):
        self.pages, self.page, self.cols = pages, page, cols
        self.table = np.full((slots, cols), -1, np.int64)
        self.data = np.zeros(pages, object)  # a page's contents: any value
        for p in range(pages):
            self.data[p] = [0] * page

    def refs(self):
        r = np.zeros(self.pages, np.int64)
        for p in self.table.ravel():
            if p >= 0:
                r[p] += 1
        return r

    def reserve(self, seq, begin, end):
        r = self.refs()
        free = [p for p in range(self.pages) if r[p] == 0]
        plan = []
        for s, b, e in zip(seq, begin, end):
            if b < e:
                plan += [(s, b, j) for j in range(b // self.page, (e - 1) // self.page + 1)
                         if self.table[s, j] < 0 or r[self.table[s, j]] > 1]
        for (s, b, j), p in zip(plan, free):
            old, self.table[s, j] = self.table[s, j], p
            if old >= 0 and j == b // self.page:
                k = b % self.page
                self.data[p] = self.data[old][:k] + self.data[p][k:]
        return len(plan) <= len(free)

    def fork(self, src, dst, rows):
        t = self.table.copy()
        for s, d, n in zip(src, dst, rows):
            k = -(-max(n, 0) // self.page)
            self.table[d] = np.where(np.arange(self.cols) < k, t[s], -1)

    def release(self, seq, rows):
        for s, n in zip(seq, rows):
            self.table[s, min(self.cols, -(-max(n, 0) // self.page)):] = -1

    def compact(self):
        r = self.refs()
        live = int((r > 0).sum())
        move = dict(zip([p for p in range(live, self.pages) if r[p]], [p for p in range(live) if not r[p]]))
        for s, d in move.items():
            self.data[d] = list(self.data[s])
        for at, p in np.ndenumerate(self.table):
            self.table[at] = move.get(int(p), int(p))
        return live
