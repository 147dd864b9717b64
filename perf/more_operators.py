"""The paged 4-bit cache of compressed rows of dsv41_amd as cases that can be timed and compared: rows put into it and
read back (append), attention of single tokens and drafts over ring and cache (decode), attention of a prompt's chunk
over window rows and cache (prefill), and the operations on its pages: sequences forked with their tail made writable
(fork), sequences cut short and the pool compacted (compact), pages copied into another pool (copy).

A row of `dim` values (512, or 576 with the values in its first 512) is held as E2M1 codes, two a byte with the lower
value in the lower four bits, and an e4m3 scale for every 16 values: 256 bytes of codes and 32 of scales for the first
512 values, for 576 then 32 bytes of codes and 4 of scales of the last 64 and 12 bytes of zeros.  A pool holds pages of
`page` rows; table[s, j] is the page of rows j * page .. of sequence s, -1 where it has none; refs counts the table's
entries that name a page.  Widths, heads, ratio, selection and contexts are the benchmark configurations' and the
reference geometry's, and odd ones between."""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.abspath("deepseekv4.1-a100-custom_amd"))

own = False

DEV = "cuda:0"
BF = torch.bfloat16
W = 128   # rows of a sequence's window ring
RD = 64   # rotated columns
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _row_bytes(dim):
    return 288 if dim == 512 else 336


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step of 24 users: those whose step closes a group of four tokens write a row, latency
        dict(name="append_24", op="append", slots=24, rows=1, start=4100, dim=576, page=64, ratio=4, closing=0.3),
        # two prompts' chunks of 32K tokens, starting inside a page
        dict(name="append_16002", op="append", slots=2, rows=8001, start=77, dim=576, page=64, ratio=4, closing=1.0),
        # one user early in a conversation, the reference geometry: fewer rows than are selected
        dict(name="decode_1", op="decode", slots=1, drafts=1, rows=300, k=512, heads=64, dim=512, page=64, ratio=2),
        # four users at 128K tokens: the decode benchmark's shape
        dict(name="decode_4", op="decode", slots=4, drafts=1, rows=32768, k=2048, heads=64, dim=576, page=64, ratio=4),
        # two short prompts going on, the reference geometry, an odd number of heads
        dict(name="prefill_301", op="prefill", batch=2, s=301, prior=1000, k=512, heads=20, dim=512, page=32, ratio=2),
        # a chunk of a long prompt: the prefill benchmark's shape
        dict(name="prefill_2048", op="prefill", batch=1, s=2048, prior=65536, k=2048, heads=64, dim=576, page=64, ratio=4),
        # four samples from one prompt
        dict(name="fork_4", op="fork", parents=1, children=4, rows=8229, more=64, dim=576, page=64),
        # seven prompts with nine samples each, long ones
        dict(name="fork_63", op="fork", parents=7, children=9, rows=30011, more=500, dim=576, page=64),
        # a few users leave, some drafts are taken back
        dict(name="compact_8", op="compact", slots=8, rows=2000, gone=0.4, dim=512, page=64),
        # a night's traffic leaves: half of a large pool is free, in holes
        dict(name="compact_96", op="compact", slots=96, rows=9000, gone=0.5, dim=576, page=64),
        # a finished prompt's pages handed over to the pool of the decoding side
        dict(name="copy_129", op="copy", pages=129, pool=1024, dim=576, page=64),
        # many of them
        dict(name="copy_6001", op="copy", pages=6001, pool=8192, dim=576, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "fork", "compact", "copy"])
    dim, page = rng.choice([512, 576, 576]), rng.choice([16, 32, 64, 64, 128])
    if op == "append":
        rows = rng.choice([1, _log(rng, 2, 8192)])
        return dict(op=op, slots=_log(rng, 1, max(1, min(64, 16384 // rows))), rows=rows, start=_log(rng, 1, 40000) - 1,
                    dim=dim, page=page, ratio=rng.choice([2, 4]), closing=0.3 if rows == 1 else 1.0)
    if op == "decode":
        slots = _log(rng, 1, 16)
        return dict(op=op, slots=slots, drafts=rng.choice([1, 1, 2, 6]), rows=_log(rng, 1, 131072 // slots),
                    k=_log(rng, 16, 2048), heads=rng.choice([8, 16, 20, 64, 64, 128]), dim=dim, page=page,
                    ratio=rng.choice([2, 4]))
    if op == "prefill":
        batch, heads, k = rng.choice([1, 1, 2]), rng.choice([8, 16, 20, 64, 64, 128]), _log(rng, 16, 2048)
        most = min(2048 * 64 * 2176 // (batch * max(heads, 16) * (k + W)), 2048 // batch)
        return dict(op=op, batch=batch, s=_log(rng, 2, most), prior=rng.choice([0, _log(rng, 1, 65536)]), k=k, heads=heads,
                    dim=dim, page=page, ratio=rng.choice([2, 4]))
    if op == "fork":
        parents = _log(rng, 1, 7)
        children = _log(rng, 1, 64 // parents)
        return dict(op=op, parents=parents, children=children, rows=_log(rng, 1, 30000), more=_log(rng, 1, 1000),
                    dim=dim, page=page)
    if op == "compact":
        slots = _log(rng, 1, 96)
        return dict(op=op, slots=slots, rows=_log(rng, 10, 864000 // slots if slots > 20 else 40000),
                    gone=rng.uniform(0.1, 0.9), dim=dim, page=page)
    pool = _log(rng, 16, 8192 * 64 // page)
    return dict(op=op, pages=_log(rng, 1, pool * 3 // 4), pool=pool, dim=dim, page=page)


# ------------------------------------------------------------------------------------------------ inputs
def _pages(rows, page):
    return -(-rows // page)


def _nibbles(x):
    """Values in groups of 16 -> (codes two a byte, scale bytes): s = e4m3(max(amax, 6 * 2^-9) / 6), E2M1 of x / s; the
    quotients in 64 bits, since bf16 values over such scales often lie on a border."""
    n, d = x.shape
    b = x.double().view(n, d // 16, 16)
    six = b.new_full((), 6.0)  # (a division by a plain number is a product with its rounded reciprocal)
    s = (b.abs().amax(-1, keepdim=True).clamp_min(6 * 2.0 ** -9) / six).clamp(max=448.0).to(torch.float8_e4m3fn)
    v = (b / s.double()).clamp(-6, 6)
    a = v.abs()
    r = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    c = (r + 8 * (v < 0)).to(torch.uint8).view(n, d // 2, 2)
    return c[..., 0] | c[..., 1] << 4, s.view(torch.uint8).view(n, d // 16)


def _packed(x):
    """Rows [n, dim] -> packed rows [n, row bytes]."""
    n, d = x.shape
    out = torch.zeros(n, _row_bytes(d), dtype=torch.uint8, device=x.device)
    out[:, :256], out[:, 256:288] = _nibbles(x[:, :512])
    if d == 576:
        out[:, 288:320], out[:, 320:324] = _nibbles(x[:, 512:])
    return out


def _latents(g, n, d):
    """Compressor outputs: normed rows in which a few channels are large."""
    x = torch.randn(n, d, generator=g, device=DEV) * 0.5
    x[:, torch.randint(0, d, (d // 64,), generator=g, device=DEV)] *= 6
    return x


def _pool(g, pages, page, dim, values=True):
    rb = _row_bytes(dim)
    if not values:  # (pages that are moved as they are)
        return torch.randint(-2 ** 62, 2 ** 62, (pages, page * rb // 8), generator=g, device=DEV).view(torch.uint8).view(pages, page, rb)
    pool = torch.empty(pages * page, rb, dtype=torch.uint8, device=DEV)
    for i in range(0, pages * page, 1 << 15):
        n = min(1 << 15, pages * page - i)
        pool[i:i + n] = _packed(_latents(g, n, dim).to(BF).float())
    return pool.view(pages, page, rb)


def _tables(g, counts, pages, wide):
    """A table whose sequence s has counts[s] pages, taken from the pool in random order; with the pages' counts."""
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(counts), wide), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[order[:at].long()] = 1
    return table, refs


def _rope_tables(n):
    f = 10000.0 ** (-torch.arange(0, RD, 2, dtype=torch.float64, device=DEV) / RD)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * f
    return a.cos().float(), a.sin().float()


def _chosen(g, seen, k, n):
    """For each row of `seen` counts: k of the first `seen` cache rows at random, ascending, -1 behind the last."""
    out = torch.empty(len(seen), k, dtype=torch.int32, device=DEV)
    for i in range(0, len(seen), 256):
        c = seen[i:i + 256, None]
        key = torch.rand(len(c), n, generator=g, device=DEV).masked_fill_(torch.arange(n, device=DEV) >= c, -1.0)
        v, p = key.topk(min(k, n), dim=1)
        p = p.masked_fill(v < 0, n).sort(1).values
        out[i:i + 256] = -1
        out[i:i + 256, :p.shape[1]] = p.masked_fill(p == n, -1).to(torch.int32)
    return out


def _i64(v):
    return torch.as_tensor(v, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 6007 + 83)
    op, dim, page = case["op"], case["dim"], case["page"]
    s = dict(case=case)
    if op == "append":
        slots, n, start = case["slots"], case["rows"], case["start"]
        each = _pages(start + n, page)
        pages = slots * each
        s["table"], s["refs"] = _tables(g, [each] * slots, pages, each + 1)
        s["pool"] = torch.zeros(pages, page, _row_bytes(dim), dtype=torch.uint8, device=DEV)
        s["latent"] = _latents(g, slots * n, dim).to(BF)
        s["seq"] = torch.arange(slots, device=DEV).repeat_interleave(n)
        row = start + torch.arange(n, device=DEV).repeat(slots)
        if case["closing"] < 1:  # (a step that closes no group writes no row)
            row[torch.rand(slots * n, generator=g, device=DEV) >= case["closing"]] = -1
        s["row"] = row
        s["cos"], s["sin"] = _rope_tables((start + n) * case["ratio"])
    elif op in ("decode", "prefill"):
        h, k, ratio = case["heads"], case["k"], case["ratio"]
        slots = case["slots"] if op == "decode" else case["batch"]
        if op == "decode":
            ctx = [max(case["drafts"], case["rows"] * ratio * (slots - i) // slots + i) for i in range(slots)]
        else:
            ctx = [case["prior"] + case["s"]] * slots
        n_c = [c // ratio for c in ctx]
        counts = [_pages(c, page) for c in n_c]
        pages = sum(counts) + 3
        s["pool"] = _pool(g, pages, page, dim)
        s["table"], s["refs"] = _tables(g, counts, pages, max(counts) + 1)
        s["sink"] = torch.randn(h, generator=g, device=DEV)
        if op == "decode":
            d = case["drafts"]
            seq = torch.arange(slots, device=DEV).repeat_interleave(d)
            pos = torch.cat([torch.arange(c - d, c, device=DEV) for c in ctx])
            s.update(seq=seq, pos=pos, pmax=(_i64(ctx) - 1)[seq])
            s["q"] = torch.randn(slots * d, 1, h, dim, generator=g, device=DEV).to(BF)
            s["ring"] = (torch.randn(slots, W, dim, generator=g, device=DEV) * 0.5).to(BF)
            s["idx"] = _chosen(g, (pos + 1) // ratio, k, max(1, max(n_c))).view(slots * d, 1, k)
            s["cos"], s["sin"] = _rope_tables(max(ctx))
        else:
            n, prior = case["s"], case["prior"]
            hist = min(prior, W - 1)
            s["q"] = torch.randn(slots, n, h, dim, generator=g, device=DEV).to(BF)
            s["kv"] = (torch.randn(slots, hist + n, dim, generator=g, device=DEV) * 0.5).to(BF)
            at = hist + torch.arange(n, device=DEV)[:, None]
            win = (at - W + 1).clamp_min(0) + torch.arange(min(W, hist + n), device=DEV)
            s["win"] = torch.where(win <= at, win, -1).to(torch.int32).expand(slots, -1, -1).contiguous()
            seen = ((prior + torch.arange(n, device=DEV) + 1) // ratio).repeat(slots)
            s["idx"] = _chosen(g, seen, k, max(1, max(n_c))).view(slots, n, k)
            s["seq"] = torch.arange(slots, device=DEV)
    elif op == "fork":
        par, ch, rows, more = case["parents"], case["children"], case["rows"], case["more"]
        each = _pages(rows, page)
        new = par * ch * (_pages(rows + more, page) - rows // page)
        pages = par * each + new + 5
        s["pool"] = _pool(g, pages, page, dim, values=False)
        table, refs = _tables(g, [each] * par + [0] * (par * ch), pages, _pages(rows + more, page))
        s["src"] = torch.arange(par, device=DEV).repeat_interleave(ch)
        s["dst"] = par + torch.arange(par * ch, device=DEV)
        s["rows"] = torch.full((par * ch,), rows, device=DEV)
        s["end"] = s["rows"] + more
        s["start"] = (table, refs)
        s["table"], s["refs"] = table.clone(), refs.clone()
    elif op == "compact":
        slots, rows = case["slots"], case["rows"]
        counts = [_pages(max(1, rows * (3 + i % 5) // 7), page) for i in range(slots)]
        pages = sum(counts) + 7
        s["pool"] = _pool(g, pages, page, dim, values=False)
        table, refs = _tables(g, counts, pages, max(counts))
        left = torch.rand(slots, generator=g, device=DEV) >= case["gone"]
        cut = torch.rand(slots, generator=g, device=DEV)  # (of those that stay a few rows are taken back)
        full = _i64(counts) * page
        s["seq"] = torch.randperm(slots, generator=g, device=DEV)
        s["rows"] = torch.where(left, full - (cut * page * 1.5).long().clamp(max=page), torch.zeros_like(full))[s["seq"]]
        s["start"] = (table, refs)
        s["table"], s["refs"] = table.clone(), refs.clone()
    else:
        n, pages = case["pages"], case["pool"]
        s["from"] = _pool(g, pages, page, dim, values=False)
        s["pool"] = _pool(g, pages, page, dim, values=False)
        s["table"], s["refs"] = _tables(g, [0], pages, 1)
        s["src"] = torch.randperm(pages, generator=g, device=DEV)[:n]
        s["dst"] = torch.randperm(pages, generator=g, device=DEV)[:n]
    if own:
        from dsv41_amd.kv4 import PagedKV4
        s["cache"] = PagedKV4(s["pool"], s["table"], s["refs"], dim=dim)
        if op == "copy":
            s["other"] = PagedKV4(s["from"], s["table"].clone(), s["refs"].clone(), dim=dim)
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _values(rows, dim):
    """Packed rows [..., row bytes] -> fp32 values [..., dim]."""
    lut = torch.tensor(E2M1 + [-v for v in E2M1], device=rows.device)

    def part(codes, scales):
        c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        return lut[c.int()] * scales.contiguous().view(torch.float8_e4m3fn).float().repeat_interleave(16, -1)
    v = part(rows[..., :256], rows[..., 256:288])
    return v if dim == 512 else torch.cat((v, part(rows[..., 288:320], rows[..., 320:324])), -1)


def _gather(pool, table, seq, row):
    """The packed rows `row` of sequences `seq` (zeros where row is -1) and which of them there are."""
    page = pool.shape[1]
    there = row >= 0
    r = row.clamp_min(0).long()
    p = table[seq, r // page].long()
    there = there & (p >= 0)
    return pool[p.clamp_min(0), r % page] * there.unsqueeze(-1), there


def _rotated(x, cos, sin, pos, sign):
    """The last RD columns of x [n, ..., d] as pairs turned by the angle of position pos [n], in 64 bits."""
    y = x.double()
    shape = (len(pos),) + (1,) * (x.dim() - 2) + (RD // 2,)
    c, s = cos[pos].double().view(shape), sign * sin[pos].double().view(shape)
    a, b = y[..., -RD::2].clone(), y[..., -RD + 1::2].clone()
    y[..., -RD::2], y[..., -RD + 1::2] = a * c - b * s, a * s + b * c
    return y


def _attend(q, k, there, sink, scale):
    """q [n, h, d], k [n, t, d] fp32, there [n, t] -> softmax over the rows that there are and the sink, times rows[:512]."""
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    x = x.masked_fill(~there[:, None], float("-inf"))
    m = torch.maximum(x.amax(-1), sink).unsqueeze(-1)
    p = torch.exp(x - m)
    den = p.sum(-1, keepdim=True) + torch.exp(sink[:, None] - m)
    return torch.matmul(p, k[..., :512].contiguous()) / den


def _ring_rows(pos, pmax):
    """Which slots of the ring a query at pos sees (nothing newer than itself): [n, W]."""
    held = pmax[:, None] - torch.remainder(pmax[:, None] - torch.arange(W, device=DEV), W)
    return (held >= 0) & (held <= pos[:, None]) & (pos[:, None] - held < W)


def _plain_attention(s):
    c, dim = s["case"], s["case"]["dim"]
    scale = dim ** -0.5
    if c["op"] == "decode":
        rows, there = _gather(s["pool"], s["table"], s["seq"][:, None], s["idx"][:, 0])
        k = torch.cat((s["ring"][s["seq"]].float(), _values(rows, dim)), 1)
        there = torch.cat((_ring_rows(s["pos"], s["pmax"]), there), 1)
        o = _attend(s["q"][:, 0].float(), k, there, s["sink"], scale)
        return dict(o=(_rotated(o, s["cos"], s["sin"], s["pos"], -1.0) if dim == 512 else o).to(BF).unsqueeze(1))
    q, win, idx = (s[n].flatten(0, 1) for n in ("q", "win", "idx"))
    batch = torch.arange(len(q), device=DEV) // s["q"].shape[1]
    out = torch.empty(*q.shape[:2], 512, dtype=BF, device=DEV)
    for i in range(0, len(q), 256):  # (the gathered rows of all queries at once would be 10 GB)
        sl = slice(i, i + 256)
        rows, there = _gather(s["pool"], s["table"], s["seq"][batch[sl], None], idx[sl])
        seen = win[sl] >= 0
        near = s["kv"][batch[sl, None], win[sl].clamp_min(0).long()].float()
        k = torch.cat((near, _values(rows, dim)), 1)
        out[sl] = _attend(q[sl].float(), k, torch.cat((seen, there), 1), s["sink"], scale).to(BF)
    return dict(o=out.view(*s["q"].shape[:3], 512))


def _named(table, seq, keep):
    """table's entries of sequences `seq` where keep, with the number of times that each counts (clamped, 1 or 0)."""
    t = table[seq]
    return t.clamp_min(0).long().flatten(), ((t >= 0) & keep).to(torch.int32).flatten()


def _plain_fork(s):
    table, refs = (t.clone() for t in s["start"])
    pool, (pages, page) = s["pool"], s["pool"].shape[:2]
    src, dst, rows, end = s["src"], s["dst"], s["rows"], s["end"]
    col = torch.arange(table.shape[1], device=DEV)
    # the fork: the destination's entries go, the source's pages of the first `rows` rows are named once more
    at, one = _named(table, dst, torch.ones_like(table[dst], dtype=torch.bool))
    refs.index_add_(0, at, -one)
    kept = col * page < rows[:, None]
    at, one = _named(table, src, kept)
    refs.index_add_(0, at, one)
    table[dst] = torch.where(kept, table[src], -1)
    # rows .. end made writable: where there is no page, or one that others name too, the lowest free page instead
    now = table[dst]
    need = (col >= rows[:, None] // page) & (col * page < end[:, None])
    need &= (now < 0) | (refs[now.clamp_min(0).long()] > 1)
    free = torch.argsort((refs > 0).to(torch.uint8), stable=True)
    new = free[(need.flatten().int().cumsum(0) - 1).clamp_min(0).long()].view(need.shape)
    at, one = now.clamp_min(0).long().flatten(), (need & (now >= 0)).to(torch.int32).flatten()
    refs.index_add_(0, at, -one)
    refs.index_add_(0, new.flatten(), need.to(torch.int32).flatten())
    table[dst] = torch.where(need, new.to(torch.int32), now)
    # what the first of these pages held before `rows` goes with it
    first = (rows // page).clamp(max=table.shape[1] - 1)
    i = torch.arange(len(dst), device=DEV)
    moved = need[i, first] & (now[i, first] >= 0)
    held = (torch.arange(page, device=DEV) < (rows % page)[:, None]) & moved[:, None]
    a, r = held.nonzero(as_tuple=True)
    pool[new[a, first[a]], r] = pool[now[a, first[a]].long(), r]
    return dict(table=table, refs=refs, pool=pool.view(pages, -1).view(torch.int64))


def _plain_compact(s):
    table, refs = (t.clone() for t in s["start"])
    pool, (pages, page) = s["pool"], s["pool"].shape[:2]
    col = torch.arange(table.shape[1], device=DEV)
    gone = col * page >= s["rows"][:, None]
    at, one = _named(table, s["seq"], gone)
    refs.index_add_(0, at, -one)
    table[s["seq"]] = torch.where(gone, -1, table[s["seq"]])
    live = refs > 0
    n = live.sum()
    ids = torch.arange(pages, device=DEV)
    src, dst = (live & (ids >= n)).nonzero()[:, 0], (~live & (ids < n)).nonzero()[:, 0]
    pool[dst] = pool[src]
    to = ids.clone()
    to[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    table = torch.where(table >= 0, to[table.clamp_min(0).long()].to(torch.int32), -1)
    return dict(live=n.to(torch.int32).view(1), table=table, refs=refs, pool=pool.view(pages, -1).view(torch.int64))


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "append":
        y = _rotated(s["latent"], s["cos"], s["sin"], s["row"].clamp_min(0) * c["ratio"], 1.0).to(BF).float()
        packed, page = _packed(y), s["pool"].shape[1]
        i = (s["row"] >= 0).nonzero()[:, 0]
        seq, row = s["seq"][i], s["row"][i]
        s["pool"][s["table"][seq, row // page].long(), row % page] = packed[i]
        return dict(values=_values(_gather(s["pool"], s["table"], s["seq"], s["row"])[0], c["dim"]).to(BF))
    if op in ("decode", "prefill"):
        return _plain_attention(s)
    if op == "fork":
        return _plain_fork(s)
    if op == "compact":
        return _plain_compact(s)
    s["pool"][s["dst"]] = s["from"][s["src"]]
    return dict(pool=s["pool"].view(s["pool"].shape[0], -1).view(torch.int64))


# ------------------------------------------------------------------------------------------------ a pass
def run(s):
    if not own:
        return _plain(s)
    from dsv41_amd.kv4 import sattn4, sparse_attn4
    c, op, cache = s["case"], s["case"]["op"], s["cache"]
    if op == "append":
        cache.append(s["latent"], s["seq"], s["row"], c["ratio"], s["cos"], s["sin"], RD)
        return dict(values=cache.read(s["seq"], s["row"]))
    if op == "decode":
        return dict(o=sattn4(s["q"], s["ring"], cache, s["idx"], s["pos"], s["sink"], s["cos"], s["sin"],
                             RD if c["dim"] == 512 else 0, c["dim"] ** -0.5, s["seq"], s["pmax"], d_v=512))
    if op == "prefill":
        return dict(o=sparse_attn4(s["q"], s["kv"], cache, s["sink"], s["win"], s["idx"], c["dim"] ** -0.5, seq=s["seq"],
                                   d_v=512))
    whole = s["pool"].view(s["pool"].shape[0], -1).view(torch.int64)
    if op == "copy":
        cache.copy_pages(s["other"], s["src"], s["dst"])
        return dict(pool=whole)
    cache.table.copy_(s["start"][0])  # (every pass starts from the same pages)
    cache.refs.copy_(s["start"][1])
    if op == "fork":
        cache.fork(s["src"], s["dst"], s["rows"])
        cache.reserve(s["dst"], s["rows"], s["end"])
        return dict(table=cache.table, refs=cache.refs, pool=whole)
    cache.release(s["seq"], s["rows"])
    live = cache.compact()
    return dict(live=live, table=cache.table, refs=cache.refs, pool=whole)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, dim, page = case["op"], case["dim"], case["page"]
    rb = _row_bytes(dim)
    if op == "append":
        n = case["slots"] * case["rows"]
        held = n * case["closing"]
        return dict(bytes=held * (2 * dim + 2 * rb) + n * (2 * dim + 16), flops=20 * held * dim)
    if op == "decode":
        rows = case["slots"] * case["drafts"]
        seen = [max(case["drafts"], case["rows"] * case["ratio"] * (case["slots"] - i) // case["slots"] + i) // case["ratio"]
                for i in range(case["slots"])]
        keys = sum(min(case["k"], n) for n in seen) * case["drafts"]
        read = sum(min(min(case["k"], n) * case["drafts"], n) for n in seen)
        ring = case["slots"] * W
        return dict(bytes=read * rb + ring * 2 * dim + rows * (case["heads"] * 2 * (dim + 512) + 4 * case["k"]),
                    flops=2 * (keys + rows * W) * case["heads"] * (dim + 512))
    if op == "prefill":
        b, n, h = case["batch"], case["s"], case["heads"]
        hist = min(case["prior"], W - 1)
        keys = sum(min(case["k"], (case["prior"] + i + 1) // case["ratio"]) + min(W, hist + i + 1) for i in range(n))
        read = min(n * case["k"], (case["prior"] + n) // case["ratio"])
        return dict(bytes=b * (read * rb + (hist + n) * 2 * dim + n * (h * 2 * (dim + 512) + 4 * case["k"] + 4 * W)),
                    flops=2 * b * keys * h * (dim + 512))
    pb = page * rb
    if op == "fork":
        n = case["parents"] * case["children"]
        col = _pages(case["rows"] + case["more"], page)
        return dict(bytes=n * (2 * (case["rows"] % page) * rb + 12 * col) + 4 * case["parents"] * col, flops=0)
    if op == "compact":
        each = sum(_pages(max(1, case["rows"] * (3 + i % 5) // 7), page) for i in range(case["slots"]))
        left = each * (1 - case["gone"])
        return dict(bytes=2 * pb * left * case["gone"] + 20 * each, flops=0)
    return dict(bytes=2 * pb * case["pages"] + 16 * case["pages"], flops=0)


# ------------------------------------------------------------------------------------------------ 64 bits
def _byte_values():
    """The two E2M1 values of each of the 256 bytes, and the e4m3 value of each."""
    def e2m1(c):
        e, f = c >> 1 & 3, c & 1
        v = f / 2 if e == 0 else (1 + f / 2) * 2.0 ** (e - 1)
        return -v if c & 8 else v

    def e4m3(b):
        e, f = b >> 3 & 15, b & 7
        v = math.nan if b & 127 == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        return -v if b & 128 else v
    two = torch.tensor([[e2m1(b & 15), e2m1(b >> 4)] for b in range(256)], dtype=torch.float64, device=DEV)
    return two, torch.tensor([e4m3(b) for b in range(256)], dtype=torch.float64, device=DEV)


def _row64(packed, dim):
    two, one = _byte_values()
    b = packed.long()
    out = torch.empty(*b.shape[:-1], dim, dtype=torch.float64, device=DEV)
    spans = [(0, 256, 288, 0, 512)] + ([(288, 320, 324, 512, 576)] if dim == 576 else [])
    for c0, c1, e, v0, v1 in spans:
        v = two[b[..., c0:c1]].reshape(*b.shape[:-1], (v1 - v0) // 16, 16)
        out[..., v0:v1] = (v * one[b[..., c1:e]].unsqueeze(-1)).flatten(-2)
    return out


def _grid64(y):
    """Values of 16-groups of y put on the grid: the nearest E2M1 (ties to even) over the group's e4m3 scale."""
    z = y.unflatten(-1, (-1, 16))
    t = torch.clamp(z.abs().amax(-1, keepdim=True), min=6 / 512) / torch.full((1,), 6.0, dtype=torch.float64, device=DEV)
    powers = torch.tensor([2.0 ** i for i in range(-9, 128)], dtype=torch.float64, device=DEV)
    step = powers[(torch.frexp(t).exponent.long() + 5).clamp_min(0)]  # (eight steps from a power of two to the next)
    t = torch.clamp(torch.round(t / step) * step, max=448)
    z = torch.clamp(z / t, -6, 6)
    step = torch.where(z.abs() < 2, 0.5, torch.where(z.abs() < 4, 1.0, 2.0))
    return (torch.round(z / step) * step * t).flatten(-2)


def _turn64(x, angle_cos, angle_sin):
    """Pairs of the last RD columns as complex numbers times cos + i sin."""
    head, tail = x[..., :-RD], x[..., -RD:]
    z = torch.view_as_complex(tail.unflatten(-1, (-1, 2)).contiguous()) * torch.complex(angle_cos, angle_sin)
    return torch.cat((head, torch.view_as_real(z).flatten(-2)), -1)


def _softmax64(q, rows, ok, sink, scale):
    x = torch.einsum("hd,td->ht", q, rows[ok]) * scale
    x = torch.cat((x, sink.double()[:, None]), 1).softmax(1)[:, :-1]
    return x @ rows[ok][:, :512]


def exact(case, seed):
    op, dim = case["op"], case["dim"]
    if op not in ("append", "decode", "prefill"):
        return None  # (pages and whole numbers)
    s = prepare(case, seed)
    if op == "append":
        at = s["row"].clamp_min(0) * case["ratio"]
        y = _turn64(s["latent"].double(), s["cos"][at].double(), s["sin"][at].double())
        y = _grid64(y.to(BF).double())  # (the cache's grid is that of bf16 rows)
        return dict(values=y * (s["row"] >= 0)[:, None])
    page = s["pool"].shape[1]

    def cache_rows(seq, idx):
        i = idx.clamp_min(0).long()
        p = s["table"][seq].long()[torch.div(i, page, rounding_mode="floor")]
        return _row64(s["pool"][p.clamp_min(0), i % page], dim), (idx >= 0) & (p >= 0)
    if op == "decode":
        out = []
        for b in range(len(s["q"])):
            e, pos, top = int(s["seq"][b]), int(s["pos"][b]), int(s["pmax"][b])
            held = [top - (top - j) % W for j in range(W)]
            seen = torch.tensor([0 <= t <= pos and pos - t < W for t in held], device=DEV)
            rows, ok = cache_rows(e, s["idx"][b, 0])
            o = _softmax64(s["q"][b, 0].double(), torch.cat((s["ring"][e].double(), rows)), torch.cat((seen, ok)), s["sink"],
                           dim ** -0.5)
            out.append(_turn64(o, s["cos"][pos].double(), -s["sin"][pos].double()) if dim == 512 else o)
        return dict(o=torch.stack(out).unsqueeze(1))
    out = torch.empty(*s["q"].shape[:3], 512, dtype=torch.float64, device=DEV)
    for e in range(out.shape[0]):
        for i in range(out.shape[1]):
            rows, ok = cache_rows(e, s["idx"][e, i])
            w = s["win"][e, i]
            k = torch.cat((s["kv"][e][w.clamp_min(0).long()].double(), rows))
            out[e, i] = _softmax64(s["q"][e, i].double(), k, torch.cat((w >= 0, ok)), s["sink"], dim ** -0.5)
    return dict(o=out)
