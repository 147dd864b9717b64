"""Compressed rows held in 4 bits, in pages, and the attention over them.

The compressed rows of the path (cache.write_compress_kv, cache.append_compressed_decode) are values on the FP4 grid --
E2M1 times an e4m3 scale per 16 -- stored in bf16.  PagedKV4 holds them as the grid's own bits, 288 bytes a row of 512
values and 336 a row of 576 instead of 1024 and 1152, in pages that sequences share:

  c = PagedKV4.empty(pages, slots, cap, dim)
  c.reserve(seq, begin, end)             pages of their own for rows begin .. end - 1 (a shared page's rows before begin copied)
  c.append(latent, seq, row, ratio, cos, sin, rd)      (append_decode: the rows by the tokens' positions)
  o = sattn4(q, ring, c, idx, ...)       decode: fused2.sattn2 with the cache in the place of kv_c
  o = sparse_attn4(q, kv, c, sink, win_idxs, topk_idxs, scale)     prefill: kernels.sparse_attn with kv2 in 4 bits
  c.fork(src, dst, rows)                 dst goes on from src's first rows (a prefix, samples of one prompt, drafts)
  c.release(seq, rows)                   the pages behind the first rows are given up
  c.compact()                            the live pages to the front of the pool
  c.copy_pages(other, src, dst)          pages out of another pool

Every call is asynchronous on the current stream, synchronises with nothing and may be captured; calls on one cache must
be stream-ordered.  Index arguments are tensors or lists (captured calls: tensors on the GPU); host memory may be filled
anew when a call returns (many entries that are not in pinned memory are waited for).  What a call that writes (append,
reserve, fork, release, compact, copy_pages) cannot do on the device -- too few free pages, an index out of range, a row
without a page -- it leaves out and notes in the cache's error word, which check() raises for (every such call does with
DSV41_CHECK_ERRORS=1).  To read and to the attentions a row that is not there is none: zeros, no key, no note.

A PagedKV4 is a handle to keep: making one checks its tensors and clears an error word (a few launches' time).

Forward only, as everything here."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import as_f32, lib, ptr, to_i64
from .a8 import _aligned, _index, _launch, _no_grad

ROW_BYTES = {512: 288, 576: 336}
PAGES = (16, 32, 64, 128, 256)
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_ERRORS = ((1, "too few free pages"), (2, "an entry was left out (an index out of range, or one named twice)"),
           (4, "a row was dropped (no page of the sequence's own there, or no rope angle)"))
_MOST_ENTRIES = 4096
_FEW_COPIES = 16384  # pairs up to which a copy needs no workspace
_I64, _I32, _BF16 = torch.int64, torch.int32, torch.bfloat16
_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class _Cache(ctypes.Structure):
    """dsv41_kv4 of include/dsv41_hip.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("pool", "table", "refs", "err")] +
                [(n, ctypes.c_int) for n in ("pages", "page", "slots", "cols", "dim")])


class PagedKV4:
    """pool uint8 [pages, page, row bytes]: per row 256 bytes of E2M1 codes (two a byte, the lower value in the lower four
    bits) and 32 e4m3 scales, one per 16 values; for 576 values then 32 bytes of codes and 4 of scales of the last 64 and
    12 zeros.  table int32 [slots, cols]: the page of rows j * page .. of a sequence, -1 none.  refs int32 [pages]: how
    many entries of the table name a page, 0: free.  The caller owns the tensors (contiguous, one GPU); dim: 512, or 576
    with the values in the first 512 columns."""

    def __init__(self, pool: torch.Tensor, table: torch.Tensor, refs: torch.Tensor, dim: int = 576):
        if dim not in ROW_BYTES:
            raise ValueError(f"PagedKV4: rows of {dim} (512 or 576)")
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[1] not in PAGES or pool.shape[2] != ROW_BYTES[dim]:
            raise ValueError(f"PagedKV4: pool {tuple(pool.shape)} {pool.dtype} (uint8 [pages, 16 to 256, {ROW_BYTES[dim]}])")
        if table.dtype != torch.int32 or table.dim() != 2 or refs.dtype != torch.int32 or refs.shape != pool.shape[:1]:
            raise ValueError(f"PagedKV4: table {tuple(table.shape)} {table.dtype}, refs {tuple(refs.shape)} {refs.dtype} "
                             f"(int32 [slots, columns] and [{pool.shape[0]}])")
        if 0 in pool.shape or 0 in table.shape or table.numel() > (1 << 31) - (1 << 20) or pool.shape[0] * pool.shape[1] >= 1 << 31:
            raise ValueError(f"PagedKV4: pool {tuple(pool.shape)}, table {tuple(table.shape)}")
        if not (pool.is_contiguous() and table.is_contiguous() and refs.is_contiguous()) or pool.data_ptr() % 16:
            raise ValueError("PagedKV4: contiguous tensors, the pool 16-byte aligned")
        self.index = _index(pool, table, refs)
        self.device = torch.device("cuda", self.index)
        self._pool, self._table, self._refs, self.dim = pool, table, refs, dim
        self.pages, self.page = pool.shape[:2]
        self.slots, self.cols = table.shape
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = _Cache(pool.data_ptr(), table.data_ptr(), refs.data_ptr(), self.err.data_ptr(), self.pages, self.page,
                         self.slots, self.cols, dim)
        self._at = ctypes.addressof(self._c)
        self._span = pool.data_ptr(), pool.data_ptr() + pool.numel()
        self._sizes = {}

    @classmethod
    def empty(cls, pages: int, slots: int, cap: int, dim: int = 576, page: int = 64, device="cuda") -> "PagedKV4":
        """A cache of `pages` free pages for `slots` sequences of up to `cap` rows."""
        if dim not in ROW_BYTES or page not in PAGES or pages < 1 or slots < 1 or cap < 1:
            raise ValueError(f"PagedKV4: {pages} pages of {page} rows of {dim}, {slots} sequences of {cap} rows")
        return cls(torch.zeros(pages, page, ROW_BYTES[dim], dtype=torch.uint8, device=device),
                   torch.full((slots, -(-cap // page)), -1, dtype=torch.int32, device=device),
                   torch.zeros(pages, dtype=torch.int32, device=device), dim)

    # (what the calls work on is fixed: the tensors' contents change, the tensors do not)
    pool = property(lambda self: self._pool)
    table = property(lambda self: self._table)
    refs = property(lambda self: self._refs)

    def _i64(self, name: str, t, n: int) -> torch.Tensor:
        """n index entries as contiguous int64 on the cache's GPU (from a tensor or a list)."""
        if not isinstance(t, torch.Tensor):
            t = torch.as_tensor(t)
            t = t.to(_I64) if t.numel() == 0 else t
        if t.numel() != n:
            raise RuntimeError(f"{name}: {t.numel()} entries beside {n}")
        if t.dtype is not _I64 or t.get_device() != self.index or not t.is_contiguous():
            if t.dtype not in _INTEGERS:
                raise RuntimeError(f"{name}: entries of {t.dtype} (integers)")
            if not t.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{name}: entries in host memory in a captured call (a replay would read them again)")
            t = to_i64(t, self.device)
        return t

    def _size(self, rows: int, h: int, wt: int, t: int, b: int) -> int:
        """Workspace bytes of an attention call."""
        key = (rows, h, wt, t, b)
        n = self._sizes.get(key)
        if n is None:
            if len(self._sizes) > 1024:
                self._sizes.clear()
            n = self._sizes[key] = lib().dsv41_kv4_attn_workspace_bytes(self._at, *key)
        return n

    def _done(self) -> None:
        if _lib.CHECK_ERRORS:
            self.check()

    def check(self) -> None:
        """Raise RuntimeError when a call left something out since the last check; clears the word.  Synchronises."""
        v = int(self.err.item())
        if v:
            self.err.zero_()
            raise RuntimeError("PagedKV4: " + "; ".join(t for bit, t in _ERRORS if v & bit))

    # ---- rows
    def append(self, latent: torch.Tensor, seq, row, ratio: int, cos: torch.Tensor, sin: torch.Tensor, rd: int) -> None:
        """latent [..., dim] bf16 (compressor outputs), one to row[i] of sequence seq[i] each (row -1: none, as in a decode
        step that closes no group): its last rd columns rotated by the angle of position row * ratio, rounded to bf16 and
        put on the 4-bit grid, as the bf16 tables' appends do.  The rows' pages must be the sequences' own (reserve); the
        rows of one call must differ."""
        self._append(latent, seq, row, ratio, 0, cos, sin, rd)

    def append_decode(self, latent: torch.Tensor, seq, pos, ratio: int, cos: torch.Tensor, sin: torch.Tensor,
                      rd: int) -> None:
        """append of a decode step (dsv41/decode.py:157-164): latent[i] to the row of the group that position pos[i] closes,
        row (pos[i] + 1) / ratio - 1; positions that close none, or are not in 0 .. 2^31 - 1, leave the cache alone (no spare
        row)."""
        self._append(latent, seq, pos, ratio, 1, cos, sin, rd)

    def _append(self, latent, seq, row, ratio: int, by_pos: int, cos, sin, rd: int) -> None:
        dim = self.dim
        if latent.shape[-1] != dim or latent.dtype != torch.bfloat16:
            raise RuntimeError(f"kv4.append: latent {tuple(latent.shape)} {latent.dtype} (bf16 rows of {dim})")
        if ratio < 1 or rd < 0 or rd > dim or rd % 2:
            raise RuntimeError(f"kv4.append: ratio {ratio}, {rd} rotated columns")
        _no_grad("kv4.append", latent)
        index = _index(self.pool, latent)
        x = latent if latent.dim() == 2 else latent.reshape(-1, dim)
        n, stride = x.shape[0], x.stride(0)
        if n == 1:
            stride = dim
        if x.stride(1) != 1 or stride % 8 or stride < dim or x.data_ptr() % 16:
            x, stride = _aligned(x.contiguous()), dim
        seq, row = self._i64("kv4.append", seq, n), self._i64("kv4.append", row, n)
        cos, sin = _angles("kv4.append", cos, sin, rd, index)
        _launch("dsv41_kv4_append", index, self._at, x.data_ptr(), stride, seq.data_ptr(), row.data_ptr(), n, ratio, by_pos,
                ptr(cos), ptr(sin), cos.shape[0] if rd else 0, rd)
        self._done()

    def read(self, seq, row) -> torch.Tensor:
        """Rows row[i] of sequences seq[i] as bf16 [..., dim] (the shape of row; exact), zeros where there is none."""
        shape = row.shape if isinstance(row, torch.Tensor) else (len(row),)
        out = torch.empty(*shape, self.dim, dtype=_BF16, device=self.device)
        n = out.numel() // self.dim
        seq, row = self._i64("kv4.read", seq, n), self._i64("kv4.read", row, n)
        _launch("dsv41_kv4_read", self.index, self._at, seq.data_ptr(), row.data_ptr(), n, out.data_ptr())
        return out

    # ---- pages
    def reserve(self, seq, begin, end) -> None:
        """Rows begin[i] .. end[i] - 1 of sequence seq[i] made writable: a page of its own wherever it has none or shares
        one, the lowest free pages in the order of the arguments.  Where a shared page is replaced its rows before begin[i]
        are copied, and no others: the rest of the page, from end[i] on too, holds what the new page held until rows are
        appended there (a sequence that goes on reserves from its length on).  Distinct sequences, 4096 at most."""
        n = _count(seq)
        if n > _MOST_ENTRIES:
            raise RuntimeError(f"kv4.reserve: {n} sequences (at most {_MOST_ENTRIES})")
        seq, begin, end = (self._i64("kv4.reserve", t, n) for t in (seq, begin, end))
        size = 4 * (self.slots + 3 * self.pages + 2 * n)
        ws = torch.empty(size // 4, dtype=_I32, device=self.device)
        _launch("dsv41_kv4_reserve", self.index, self._at, seq.data_ptr(), begin.data_ptr(), end.data_ptr(), n,
                ws.data_ptr(), size)
        self._done()

    def fork(self, src, dst, rows=None) -> None:
        """Sequence dst[i] gets the first rows[i] rows (None: all) of src[i] in place of its own, by naming their pages:
        nothing is copied before reserve makes a shared page writable.  A destination may be named once and may not be a
        source of the same call."""
        n = _count(src)
        _launchable("kv4.fork", n)
        src, dst = self._i64("kv4.fork", src, n), self._i64("kv4.fork", dst, n)
        rows = None if rows is None else self._i64("kv4.fork", rows, n)
        _launch("dsv41_kv4_fork", self.index, self._at, src.data_ptr(), dst.data_ptr(), ptr(rows), n)
        self._done()

    def release(self, seq, rows=None) -> None:
        """The pages behind the first rows[i] rows (None: 0, all of them) of sequence seq[i] are given up."""
        n = _count(seq)
        _launchable("kv4.release", n)
        seq = self._i64("kv4.release", seq, n)
        rows = None if rows is None else self._i64("kv4.release", rows, n)
        _launch("dsv41_kv4_release", self.index, self._at, seq.data_ptr(), ptr(rows), n)
        self._done()

    def compact(self) -> torch.Tensor:
        """The live pages moved to the front of the pool (those that stand there stay); table and refs follow.  Returns how
        many they are, int32 [1] on the GPU: the pool's pages behind them are free.  The counts have to be the table's: an
        entry behind the live pages whose page has none is taken out and noted."""
        size = 4 * (2 + 3 * self.pages)
        ws = torch.empty(size // 4, dtype=_I32, device=self.device)
        live = torch.empty(1, dtype=_I32, device=self.device)
        _launch("dsv41_kv4_compact", self.index, self._at, live.data_ptr(), ws.data_ptr(), size)
        self._done()
        return live

    def copy_pages(self, other: "PagedKV4", src, dst) -> None:
        """Pages src[i] of another cache's pool into this pool's pages dst[i] (-1: none): contents alone, no table.  Both
        pools have rows and pages of one size and stand on one GPU; where a destination is named twice the last pair has
        it."""
        if other.dim != self.dim or other.page != self.page:
            raise RuntimeError(f"kv4.copy_pages: pages of {other.page} rows of {other.dim} into {self.page} of {self.dim}")
        if other.index != self.index:
            raise RuntimeError(f"kv4.copy_pages: pools on {other.device}, {self.device}")
        if self._span[0] < other._span[1] and other._span[0] < self._span[1]:
            raise RuntimeError("kv4.copy_pages: the pools are one memory (fork and reserve share and copy within a pool)")
        n = _count(src)
        _launchable("kv4.copy_pages", n)
        src, dst = self._i64("kv4.copy_pages", src, n), self._i64("kv4.copy_pages", dst, n)
        size = 4 * self.pages if n > _FEW_COPIES else 0  # (dsv41_kv4_copy_workspace_bytes)
        ws = torch.empty(size // 4, dtype=_I32, device=self.device) if size else None
        _launch("dsv41_kv4_copy", self.index, self._at, other._at, src.data_ptr(), dst.data_ptr(), n, ptr(ws), size)
        self._done()


def _count(t) -> int:
    return t.numel() if isinstance(t, torch.Tensor) else len(t)


def _launchable(name: str, n: int) -> None:
    if n >= 1 << 24:  # (a workgroup of 256 each: 2^32 lanes)
        raise RuntimeError(f"{name}: {n} entries (at most {(1 << 24) - 1})")


def _angles(name: str, cos, sin, rd: int, index: int):
    """The rope tables [positions, rd / 2] as contiguous fp32 (None without a rotation)."""
    if rd == 0:
        return None, None
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != rd // 2:
        raise RuntimeError(f"{name}: rope tables {tuple(cos.shape)}, {tuple(sin.shape)} for {rd} columns")
    if cos.get_device() != index or sin.get_device() != index:
        raise RuntimeError(f"{name}: rope tables on {cos.device}, {sin.device}")
    return as_f32(cos), as_f32(sin)


def _operands(name: str, q, cache, sink, h: int, *more):
    """Checks that both attentions share; q contiguous and aligned, the sink."""
    if not isinstance(cache, PagedKV4):
        raise TypeError(f"{name}: a PagedKV4 expected")
    index = _index(cache.pool, q, sink, *more)
    _no_grad(name, q, sink, *more)
    if q.dtype != torch.bfloat16 or q.shape[-1] != cache.dim:
        raise RuntimeError(f"{name}: q {tuple(q.shape)} {q.dtype} (bf16 rows of {cache.dim})")
    if sink.shape != (h,):
        raise RuntimeError(f"{name}: sink {tuple(sink.shape)} for {h} heads")
    return index, _aligned(q.contiguous()), as_f32(sink)


def _window(name: str, kv: torch.Tensor, dim: int) -> torch.Tensor:
    """Window rows with unit and row strides, 16-byte aligned (a copy where they have others)."""
    if kv.dim() != 3 or kv.dtype != torch.bfloat16 or kv.shape[-1] != dim:
        raise RuntimeError(f"{name}: window rows {tuple(kv.shape)} {kv.dtype} (bf16 [., ., {dim}])")
    if kv.stride(2) != 1 or kv.stride(1) != dim or kv.stride(0) % 8 or kv.data_ptr() % 16:
        kv = _aligned(kv.contiguous())
        if kv.stride(0) % 8:  # (a batch of one has any stride)
            kv = kv.view(-1).view(kv.shape)
    return kv


def _indices(name: str, idx, shape: tuple, index: int):
    """An index list [..., t] as contiguous int32 and its t (None: 0)."""
    if idx is None:
        return None, 0
    if idx.shape[:-1] != shape or idx.get_device() != index:
        raise RuntimeError(f"{name}: indices {tuple(idx.shape)} on {idx.device} for {shape}")
    if idx.dtype not in _INTEGERS:
        raise RuntimeError(f"{name}: indices of {idx.dtype} (integers)")
    if idx.dtype == _I64:  # (the narrower types have no such values, nor room for the bounds)
        idx = idx.clamp(-1, 2 ** 31 - 1)
    idx = idx.to(torch.int32).contiguous()
    return (idx, idx.shape[-1]) if idx.shape[-1] else (None, 0)


def _values_of(name: str, d_v: int | None) -> None:
    if d_v not in (None, 512):
        raise RuntimeError(f"{name}: values of {d_v} columns (512)")


def sattn4(q, kv_win, cache: PagedKV4, idx, pos, attn_sink, cos, sin, rd: int, softmax_scale: float, seq, pmax, plim=None,
           d_v: int | None = None) -> torch.Tensor:
    """fused2.sattn2 (dsv41/fused2.py:417-446) with the compressed rows in a 4-bit cache.

    q [B, 1, h, dim] bf16 (row b at position pos[b] of sequence seq[b]); kv_win [S, win, dim] bf16 rings; idx [B, 1, t]
    cache rows of the row's sequence (-1, or without a page: none) or None; pmax [B] the newest position written to the
    row's ring, plim [B] (default pos) the newest it may see.  Returns [B, 1, h, 512] bf16 with the inverse rope on the
    last rd columns (a multiple of 4; 0: none), rounded once; a row that sees no key is zeros, a position outside the rope
    tables NaN there."""
    b, s, h, d = q.shape
    if s != 1:
        raise RuntimeError(f"sattn4: {s} tokens a row (1)")
    _values_of("sattn4", d_v)
    index, q, sink = _operands("sattn4", q, cache, attn_sink, h, kv_win)
    if rd % 4 or rd < 0 or rd > 512:
        raise RuntimeError(f"sattn4: {rd} rotated columns (a multiple of 4, at most 512)")
    cos, sin = _angles("sattn4", cos, sin, rd, index)
    kv_win = _window("sattn4", kv_win, d)
    idx, t = _indices("sattn4", idx, (b, 1), index)
    pos, seq, pmax = (cache._i64("sattn4", x, b) for x in (pos, seq, pmax))
    plim = None if plim is None else cache._i64("sattn4", plim, b)
    out = torch.empty(b, 1, h, 512, dtype=_BF16, device=cache.device)
    slots, win = kv_win.shape[:2]
    size = cache._size(b, h, win, t, 0)
    ws = torch.empty(size // 4, dtype=torch.float32, device=cache.device) if size else None
    _launch("dsv41_sattn4", index, cache._at, q.data_ptr(), kv_win.data_ptr(), kv_win.stride(0), slots, win, ptr(idx), t,
            pos.data_ptr(), seq.data_ptr(), pmax.data_ptr(), ptr(plim), sink.data_ptr(), ptr(cos), ptr(sin),
            cos.shape[0] if rd else 0, rd, softmax_scale, out.data_ptr(), b, h, ptr(ws), size)
    return out


def sparse_attn4(q, kv, cache: PagedKV4, attn_sink, win_idxs, topk_idxs, softmax_scale: float, seq=None,
                 d_v: int | None = None) -> torch.Tensor:
    """kernels.sparse_attn (dsv41/kernels.py:172-256) over [window rows | rows of a 4-bit cache].

    q [b, s, h, dim] bf16; kv [b, n, dim] bf16 window rows and win_idxs [b, s, w] into them; topk_idxs [b, s, t] rows of the
    cache's sequence seq[i] of batch row i (None: i); -1 (or past the end, or without a page) is none, and either list may
    be None.  Returns [b, s, h, 512] bf16, rounded once; a query that sees no key is zeros.  Where many queries of more than
    32 heads list more than four times the rows that the b sequences' tables have room for, these are decoded to bf16 first, in
    a workspace of 2 * dim bytes a row, mapped or not."""
    b, s, h, d = q.shape
    _values_of("sparse_attn4", d_v)
    index, q, sink = _operands("sparse_attn4", q, cache, attn_sink, h, kv)
    if kv is not None:
        kv = _window("sparse_attn4", kv, d)
        if kv.shape[0] != b:
            raise RuntimeError(f"sparse_attn4: window rows {tuple(kv.shape)} for {b} batch rows")
    win_idxs, w = _indices("sparse_attn4", win_idxs, (b, s), index)
    if w and kv is None:
        raise RuntimeError("sparse_attn4: window indices without rows")
    if kv is not None and kv.shape[1] == 0:  # (every index is past the end)
        kv, win_idxs, w = None, None, 0
    idx, t = _indices("sparse_attn4", topk_idxs, (b, s), index)
    if seq is None and b > cache.slots:
        raise RuntimeError(f"sparse_attn4: {b} batch rows over {cache.slots} sequences")
    seq = None if seq is None else cache._i64("sparse_attn4", seq, b)
    out = torch.empty(b, s, h, 512, dtype=_BF16, device=cache.device)
    size = cache._size(b * s, h, w, t, b)
    ws = torch.empty(size // 4, dtype=torch.float32, device=cache.device) if size else None
    _launch("dsv41_sparse_attn4", index, cache._at, q.data_ptr(), ptr(kv), kv.stride(0) if kv is not None else 0,
            kv.shape[1] if kv is not None else 0, ptr(win_idxs), w, ptr(idx), t, ptr(seq), sink.data_ptr(), softmax_scale,
            out.data_ptr(), b, s, h, ptr(ws), size)
    return out
