"""The 8-bit paged K/V cache of include/ct_kv8.h on torch tensors.

`Cache` and `Seqs` hold the tensors a caller owns; the methods check their
arguments and call the C entry points on the current torch stream of the
cache's device.  They never synchronise (`status` does, and `values` without `n`).

    cache = Cache.empty(n_pages, n_layers, kv_heads, head_dim, "e4m3")
    seqs = Seqs.empty(n_seqs, max_pages)
    cache.reserve(seqs, add)                            # room for this step's rows
    for layer in range(n_layers):
        cache.append(layer, seqs, k, v)                 # [n_seqs, kv_heads, head_dim], one row each
        out = cache.attend(layer, seqs, q)              # [n_seqs, heads, head_dim]
    cache.free(seqs)
"""
from __future__ import annotations

import ctypes

import torch

from . import abi

ROWS = 16                                # token rows of a page (CT_KV8_ROWS)
FORMATS = {"e4m3": 0, "int8": 1}
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


class KV8Error(RuntimeError):
    """A ct_kv8_* call returned an error code (`code`)."""

    def __init__(self, name, code):
        super().__init__(f"{name} failed: {code}")
        self.code = code


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _int32(*numbers):
    """ctypes would cut them to 32 bits without a word."""
    if max(numbers) > 0x7FFFFFFF or min(numbers) < -0x80000000:
        raise ValueError("row counts, lengths, windows and sinks: 32-bit integers")


def _ints(t, shape, device, what):
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.is_contiguous() and t.device == device
            and (shape is None or t.shape == shape)):
        raise ValueError(f"{what}: a contiguous int32 tensor" + (f" {list(shape)}" if shape is not None else "")
                         + f" on {device}")
    return t.data_ptr()


class Seqs:
    """Sequences: page table [n_seqs, max_pages] and lengths [n_seqs], int32."""

    def __init__(self, table, lens):
        _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, "table: [n_seqs, max_pages]")
        p = _ints(table, None, table.device, "table")
        q = _ints(lens, (table.shape[0],), table.device, "lens")
        self.table, self.lens = table, lens
        self.n, self.max_pages = table.shape
        self.device = table.device
        self.c = abi.KV8Seqs(p, q, self.n, self.max_pages)
        self.ref = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, n_seqs, max_pages, device="cuda"):
        return cls(torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device))


class Cache:
    """A pool of pages: codes uint8 [pages, layers, 2, kv_heads, 16, head_dim], scales float32
    [pages, layers, 2, kv_heads], refs int32 [pages] (None: the caller assigns pages itself)."""

    def __init__(self, codes, scales, refs=None, fmt="e4m3"):
        _need(codes.dtype == torch.uint8 and codes.dim() == 6 and codes.is_contiguous() and codes.is_cuda
              and codes.shape[2] == 2 and codes.shape[4] == ROWS and codes.shape[5] in (64, 128)
              and codes.data_ptr() % 16 == 0,
              "codes: a contiguous uint8 tensor [pages, layers, 2, kv_heads, 16, 64 or 128] on a GPU, 16-byte aligned")
        _need(scales.dtype == torch.float32 and scales.is_contiguous() and scales.shape == codes.shape[:4]
              and scales.device == codes.device, "scales: a contiguous float32 tensor [pages, layers, 2, kv_heads]")
        _need(fmt in FORMATS, "fmt: 'e4m3' or 'int8'")
        self.codes, self.scales, self.refs, self.fmt = codes, scales, refs, fmt
        self.n_pages, self.n_layers, _, self.kv_heads, _, self.head_dim = codes.shape
        self.device = codes.device
        self.scale = self.head_dim ** -0.5
        r = _ints(refs, (self.n_pages,), self.device, "refs") if refs is not None else None
        self.lib = abi.load()
        self.c = abi.KV8Cache(codes.data_ptr(), scales.data_ptr(), r, self.n_pages, self.n_layers, self.kv_heads,
                              self.head_dim, FORMATS[fmt])
        self.ref = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, n_pages, n_layers, kv_heads, head_dim, fmt="e4m3", device="cuda"):
        shape = (n_pages, n_layers, 2, kv_heads)
        return cls(torch.zeros(*shape, ROWS, head_dim, dtype=torch.uint8, device=device),
                   torch.zeros(*shape, device=device), torch.zeros(n_pages, dtype=torch.int32, device=device), fmt)

    # ---- helpers (short paths: a decode step's calls are a few microseconds of GPU work each)
    def _call(self, name, *args):
        """The C call with this device current, on its current torch stream."""
        index = self.device.index
        if torch._C._cuda_getDevice() == index:
            rc = getattr(self.lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = getattr(self.lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            raise KV8Error(name, rc)

    def _seqs(self, s):
        if s.device != self.device:
            raise ValueError(f"the sequences are not on {self.device}")
        return s.ref

    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer: 0 .. {self.n_layers - 1}")
        return layer

    def _rows(self, x, what):
        """Rows, heads and row stride of [rows, heads, head_dim] with each row contiguous, and its address."""
        try:
            (n, h, d), (ld, sh, sd) = x.shape, x.stride()
        except (ValueError, AttributeError):
            raise ValueError(f"{what}: [rows, heads, {self.head_dim}]") from None
        if n == 1:
            ld = h * d
        p = x.data_ptr()
        if (d != self.head_dim or n == 0 or h == 0 or sd != 1 or (sh != d and h > 1) or not h * d <= ld < 1 << 31
                or x.dtype not in _TYPES or x.device != self.device or (p | ld * x.element_size()) & 15):
            raise ValueError(f"{what}: float32 or bfloat16 [rows, heads, {self.head_dim}] on {self.device}, each row "
                             "contiguous, rows of 16-byte alignment that do not overlap, less than 2^31 elements apart")
        return n, h, ld, p

    def _ws(self, ws, need):
        """Address and size of a workspace: the caller's (the C call checks its size) or a new one of need() bytes."""
        if ws is None:
            n = need()
            if n == 0:
                return None, None, 0
            ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        elif ws.dtype != torch.uint8 or not ws.is_contiguous() or ws.device != self.device:
            raise ValueError(f"ws: a contiguous uint8 tensor on {self.device}")
        return ws, ws.data_ptr(), ws.numel()

    def _starts(self, seqs, rows, row_start, max_rows):
        if row_start is None:
            _need(max_rows == 1 and rows >= seqs.n, "without row_start: max_rows 1 and a row for each sequence")
            return None
        return _ints(row_start, (seqs.n + 1,), self.device, "row_start")

    # ---- operators
    def append(self, layer, seqs, k, v, row_start=None, max_rows=1):
        """Write the rows k, v [rows, kv_heads, head_dim] (ct_kv8_append)."""
        n, h, ldk, pk = self._rows(k, "k")
        nv, hv, ldv, pv = self._rows(v, "v")
        _need(k.dtype == v.dtype and n == nv and h == hv == self.kv_heads,
              f"k and v: the same type and number of rows, {self.kv_heads} heads")
        rs = self._starts(seqs, n, row_start, max_rows)
        _int32(max_rows)
        self._call("ct_kv8_append", self.ref, self._layer(layer), self._seqs(seqs), pk, ldk, pv, ldv,
                   _TYPES[k.dtype], n, rs, max_rows)

    def attend_workspace(self, seqs, q, max_rows=1, max_len=None, causal=True, window=0, sinks=0):
        """A workspace for `attend` calls of these sizes (one per stream that may run them at the same time)."""
        n, h, _, _ = self._rows(q, "q")
        if max_len is None:
            max_len = seqs.max_pages * ROWS
        _int32(max_rows, max_len, window, sinks)
        n = self.lib.ct_kv8_attn_ws_bytes(self.ref, seqs.ref, _TYPES[q.dtype], n, max_rows, max_len, h, int(causal),
                                          window, sinks)
        return torch.empty(max(n, 256), dtype=torch.uint8, device=self.device)

    def attend(self, layer, seqs, q, out=None, row_start=None, max_rows=1, max_len=None, causal=True, window=0,
               sinks=0, scale=None, ws=None):
        """Attention of q [rows, heads, head_dim] over the sequences' pages (ct_kv8_attn); max_len bounds their
        lengths (default: the table's width)."""
        n, h, ldq, pq = self._rows(q, "q")
        typ = _TYPES[q.dtype]
        if out is None:
            out = torch.empty((n, h, self.head_dim), dtype=q.dtype, device=self.device)
            ldo, po = h * self.head_dim, out.data_ptr()
        else:
            no, ho, ldo, po = self._rows(out, "out")
            _need(out.dtype == q.dtype and no == n and ho == h, "out: q's shape and type")
        _need(h % self.kv_heads == 0, "heads: a multiple of kv_heads")
        rs = self._starts(seqs, n, row_start, max_rows)
        if max_len is None:
            max_len = seqs.max_pages * ROWS
        _int32(max_rows, max_len, window, sinks)
        causal = int(causal)
        ws, pw, nw = self._ws(ws, lambda: self.lib.ct_kv8_attn_ws_bytes(self.ref, seqs.ref, typ, n, max_rows, max_len,
                                                                       h, causal, window, sinks))
        self._call("ct_kv8_attn", self.ref, self._layer(layer), self._seqs(seqs), pq, ldq, po, ldo, typ, n, rs,
                   max_rows, max_len, h, self.scale if scale is None else scale, causal, window, sinks, pw, nw)
        return out

    def pages_workspace(self, seqs):
        """A workspace for `reserve` and `compact` of seqs, and for `fork` into them."""
        n = self.lib.ct_kv8_pages_ws_bytes(self.ref, seqs.n)
        return torch.empty(max(n, 256), dtype=torch.uint8, device=self.device)

    def _pages_ws(self, seqs, ws):
        return self._ws(ws, lambda: self.lib.ct_kv8_pages_ws_bytes(self.ref, seqs.n))

    def reserve(self, seqs, add, ws=None):
        """lens += add, with pages for the new rows (ct_kv8_reserve)."""
        a = _ints(add, (seqs.n,), self.device, "add")
        ws, p, n = self._pages_ws(seqs, ws)
        self._call("ct_kv8_reserve", self.ref, self._seqs(seqs), a, p, n)

    def fork(self, src, parents, dst, ws=None):
        """Sequence i of dst continues src[parents[i]] (ct_kv8_fork)."""
        a = _ints(parents, (dst.n,), self.device, "parents")
        ws, p, n = self._pages_ws(dst, ws)
        self._call("ct_kv8_fork", self.ref, self._seqs(src), a, self._seqs(dst), p, n)

    def free(self, seqs, which=None):
        """Release all sequences, or those listed in which (ct_kv8_free)."""
        w = None if which is None else _ints(which, None, self.device, "which")
        p = self._seqs(seqs)
        if which is not None and which.numel() == 0:   # its address is NULL, which means all
            return
        self._call("ct_kv8_free", self.ref, p, w, 0 if which is None else which.numel())

    def trim(self, seqs, window, sinks=0):
        """Release the pages that a window has passed (ct_kv8_trim)."""
        _int32(window, sinks)
        self._call("ct_kv8_trim", self.ref, self._seqs(seqs), window, sinks)

    def compact(self, seqs, refs_out=None, table_out=None, n_live=None, ws=None):
        """Move the live pages to the pool's start (ct_kv8_compact); in place unless outputs are given."""
        _need(self.refs is not None, "the cache has no refs")
        refs_out = self.refs if refs_out is None else refs_out
        table_out = seqs.table if table_out is None else table_out
        r = _ints(refs_out, (self.n_pages,), self.device, "refs_out")
        t = _ints(table_out, tuple(seqs.table.shape), self.device, "table_out")
        k = None if n_live is None else _ints(n_live, (1,), self.device, "n_live")
        ws, p, n = self._pages_ws(seqs, ws)
        self._call("ct_kv8_compact", self.ref, self._seqs(seqs), r, t, k, p, n)

    def copy_pages(self, src, dst):
        """Copy pages src[i] -> dst[i] (ct_kv8_copy_pages)."""
        a, b = _ints(src, None, self.device, "src"), _ints(dst, None, self.device, "dst")
        _need(src.numel() == dst.numel(), "src and dst: the same number of pages")
        self._call("ct_kv8_copy_pages", self.ref, a, b, src.numel())

    def status(self):
        """Read and clear the device status word (waits for the device)."""
        with torch.cuda.device(self.device):
            return self.lib.ct_kv8_status()

    def values(self, layer, seqs, s, n=None):
        """K and V of the first n (default: all) rows of sequence s as float32 [n, kv_heads, head_dim] each;
        rows of released pages are NaN. Without n it waits for the device, to know the length."""
        n = int(seqs.lens[s]) if n is None else n
        pages = seqs.table[s, :(n + ROWS - 1) // ROWS].long()
        gone = (pages < 0) | (pages >= self.n_pages)
        pages = pages.masked_fill(gone, 0)
        x = self.codes[pages, layer].view(torch.float8_e4m3fn if self.fmt == "e4m3" else torch.int8).float()
        scales = self.scales[pages, layer].masked_fill(gone[:, None, None], float("nan"))
        x = (x * scales[..., None, None]).permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :n]
        return x[0], x[1]
