"""The 8-bit paged cache's definitions in 64 bits (include/ct_kv8.h), for its tests: plain loops over
sequences, blocks and heads on the CPU, sharing no code with the package."""
import math

import numpy as np

ROWS = 16


def pages_of(n):
    return -(-n // ROWS)


def block_scale(amax, fmt):
    """The smallest power of two (at least 2^-126) with amax / scale within the codes' range."""
    top = 448.0 if fmt == "e4m3" else 127.0
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax / top)[1] - 1)
        while amax > top * 2.0 ** e:
            e += 1
        while e > -126 and amax <= top * 2.0 ** (e - 1):
            e -= 1
    return 2.0 ** e


def nearest(y, fmt):
    """Values of the codes nearest to y, ties to even, saturating."""
    y = np.asarray(y, np.float64)
    if fmt == "int8":
        return np.clip(np.rint(y), -127, 127)
    e = np.maximum(np.frexp(np.abs(y))[1] - 1, -6)
    step = np.exp2(e - 3.0)
    with np.errstate(invalid="ignore"):
        r = np.where(np.isfinite(y), np.rint(y / step) * step, np.sign(y) * 448.0)
    return np.clip(r, -448.0, 448.0)


class Cache:
    """values [pages][layers][2][heads][16][dim] in units of scales [pages][layers][2][heads]."""

    def __init__(self, codes, scales, refs, fmt):
        self.v, self.s, self.refs, self.fmt = codes.copy(), scales.copy(), refs.copy(), fmt

    def append(self, layer, table, lens, k, v, starts):
        for q in range(len(lens)):
            n = starts[q + 1] - starts[q]
            p0 = lens[q] - n
            for b in range(p0 // ROWS, pages_of(lens[q])):
                page = table[q][b]
                lo, hi = max(p0 - b * ROWS, 0), min(lens[q] - b * ROWS, ROWS)
                r = starts[q] + b * ROWS - p0
                for kv, src in ((0, k), (1, v)):
                    for h in range(src.shape[1]):
                        x = src[r + lo:r + hi, h].astype(np.float64)
                        fin = np.abs(x[np.isfinite(x)])
                        s = block_scale(fin.max() if fin.size else 0.0, self.fmt)
                        nan = np.isnan(x).any()
                        blk, old = self.v[page, layer, kv, h], self.s[page, layer, kv, h]
                        if lo:
                            nan |= np.isnan(old)
                            s = max(s, old) if not np.isnan(old) else s
                            if old < s:
                                blk[:lo] = nearest(blk[:lo] * (old / s), self.fmt)
                        blk[lo:hi] = nearest(np.where(np.isnan(x), 0.0, x) / s, self.fmt)
                        self.s[page, layer, kv, h] = np.nan if nan else s

    def rows(self, layer, row, n, h):
        pages = row[:pages_of(n)]
        x = self.v[pages, layer, :, h] * self.s[pages, layer, :, h][..., None, None]   # [blocks, 2, 16, dim]
        return x[:, 0].reshape(-1, x.shape[-1])[:n], x[:, 1].reshape(-1, x.shape[-1])[:n]


def sees(t, j, length, causal, window, sinks):
    ok = j < length
    if causal:
        ok = ok & (j <= t)
        if window:
            ok = ok & ((j > t - window) | (j < sinks))
    return ok


def attend(cache, layer, table, lens, q, starts, heads_kv, scale, causal=True, window=0, sinks=0):
    """out, mass = sum p |v|, reach = max_j scale max|q| sum_d |k| and total = sum |v|: what a row's rounding errors
    scale with."""
    R, H, D = q.shape
    G = H // heads_kv
    out, mass, total, reach = np.zeros((R, H, D)), np.zeros((R, H, D)), np.zeros((R, H, D)), np.zeros((R, H, 1))
    for s in range(len(lens)):
        n, L = starts[s + 1] - starts[s], max(int(lens[s]), 0)
        if not L:
            continue
        for h in range(H):
            need = pages_of(L)
            row = np.where(np.asarray(table[s][:need]) < 0, 0, table[s][:need])   # released pages: never seen
            K, V = cache.rows(layer, row, L, h // G)
            x = scale * (q[starts[s]:starts[s + 1], h].astype(np.float64) @ K.T)
            t = L - n + np.arange(n)[:, None]
            see = np.broadcast_to(sees(t, np.arange(L)[None], L, causal, window, sinks), x.shape)
            some = see.any(1)
            x = np.where(see, x, -np.inf)
            with np.errstate(invalid="ignore"):
                m = np.where(some, np.nanmax(np.where(see, x, -np.inf), 1), 0.0)[:, None]
                p = np.where(see, np.exp(x - m), 0.0)
                den = p.sum(1, keepdims=True)
                p = np.divide(p, den, out=np.zeros_like(p), where=den != 0)
            r = slice(starts[s], starts[s + 1])
            for i in range(n):                       # only visible keys: what hides holds anything
                j = see[i]
                out[r.start + i, h] = p[i, j] @ V[j]
                mass[r.start + i, h] = p[i, j] @ np.abs(V[j])
                total[r.start + i, h] = np.abs(V[j]).sum(0)
            qm = np.abs(q[r, h].astype(np.float64)).max(1)
            k1 = np.abs(K).sum(1)
            reach[r, h, 0] = scale * qm * np.max(np.where(see, k1[None], 0.0), 1)
    return out, mass, reach, total


# ---- pages
def reserve(table, lens, refs, add, stride):
    """Returns whether something was left out for lack of pages, and for a bad argument."""
    free = [p for p, r in enumerate(refs) if r == 0]
    asked, none, bad = 0, False, False
    for s in range(len(lens)):
        old = max(lens[s], 0)
        if add[s] < 0 or old + add[s] > stride * ROWS:
            bad = True
            continue
        n = pages_of(old + add[s]) - pages_of(old)
        asked += n
        if n and asked > len(free):
            none = True
            continue
        for i in range(n):
            p = free[asked - n + i]
            table[s][pages_of(old) + i] = p
            refs[p] = 1
        lens[s] = old + add[s]
    return none, bad


def fork(table, lens, refs, parents, new_table, new_lens):
    """Returns the pages copied, (from, to)."""
    free = [p for p, r in enumerate(refs) if r == 0]
    asked, copies = 0, []
    for i, q in enumerate(parents):
        new_lens[i] = 0
        if q < 0 or q >= len(lens) or lens[q] <= 0 or pages_of(lens[q]) > len(new_table[i]):
            continue
        full, tail = lens[q] // ROWS, lens[q] % ROWS
        if tail:
            asked += 1
            if asked > len(free):
                continue
            new_table[i][full] = free[asked - 1]
            refs[free[asked - 1]] = 1
            copies.append((table[q][full], free[asked - 1]))
        for b in range(full):
            new_table[i][b] = table[q][b]
            if table[q][b] >= 0:
                refs[table[q][b]] += 1
        new_lens[i] = lens[q]
    return copies


def release(table, lens, refs, which):
    for s in which:
        for b in range(pages_of(max(lens[s], 0))):
            if table[s][b] >= 0:
                refs[table[s][b]] -= 1
        lens[s] = 0


def trim(table, lens, refs, window, sinks):
    for s in range(len(lens)):
        for b in range(pages_of(sinks), max(lens[s] - window, 0) // ROWS):
            if table[s][b] >= 0:
                refs[table[s][b]] -= 1
                table[s][b] = -1


def compact(table, lens, refs):
    live = [p for p, r in enumerate(refs) if r > 0]
    L = len(live)
    move = dict(zip([p for p in live if p >= L], [p for p in range(L) if refs[p] == 0]))
    new_refs = [0] * len(refs)
    for p in live:
        new_refs[move.get(p, p)] = refs[p]
    new_table = [[move.get(p, p) if b < pages_of(max(n, 0)) else p for b, p in enumerate(r)]
                 for r, n in zip(table, lens)]
    return new_table, new_refs, move, L
