"""Cases of the 8-bit paged key/value cache: writing rows into it, attention over it, and its pages.

A cache holds pages of 16 token rows, codes [pages][layers][K, V][kv heads][16][head dim] in 8 bits (E4M3 or
int8), with one power-of-two scale for each block of 16 rows and head.  A sequence is a row of a page table and a
length.  `run` makes one pass through one operator: the framework's kernels where `own` is true, elementary torch
operations otherwise.
"""
import importlib
import math
import random

import torch

own = False
ROWS = 16
NONE = -(2.0 ** 126)


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token of a single dictation stream, behind 40 others
        dict(name="append-one", op="append", fmt="int8", type="f32", layers=1, kvh=8, dim=128, seqs=1, rows_lo=1,
             rows_hi=1, past_lo=40, past_hi=40),
        # a decode step of a full slot table (256 slots), every sequence at another offset inside its page
        dict(name="append-step", op="append", fmt="e4m3", type="bf16", layers=1, kvh=8, dim=128, seqs=256, rows_lo=1,
             rows_hi=1, past_lo=10, past_hi=1000),
        # ragged prompts written in one call, some behind earlier rows of theirs
        dict(name="append-prompts", op="append", fmt="e4m3", type="bf16", layers=1, kvh=8, dim=128, seqs=24,
             rows_lo=301, rows_hi=4001, past_lo=0, past_hi=500),
        # cross attention of one 30 s utterance: 376 encoder rows, one query row
        dict(name="attend-one", op="attend", fmt="int8", type="f32", layers=1, heads=8, kvh=8, dim=128, seqs=1,
             rows_lo=1, rows_hi=1, past_lo=375, past_hi=375, causal=False, window=0, sinks=0),
        # a decode step of 64 ragged sequences in the decoder's own head layout
        dict(name="attend-step", op="attend", fmt="e4m3", type="f32", layers=1, heads=8, kvh=8, dim=128, seqs=64,
             rows_lo=1, rows_hi=1, past_lo=60, past_hi=1023, causal=True, window=0, sinks=0),
        # long contexts with shared heads, one token each
        dict(name="attend-long", op="attend", fmt="e4m3", type="bf16", layers=1, heads=32, kvh=8, dim=128, seqs=16,
             rows_lo=1, rows_hi=1, past_lo=8000, past_hi=65000, causal=True, window=0, sinks=0),
        # streams that never end: the last 2048 keys and the first 4, a few tokens at a time
        dict(name="attend-stream", op="attend", fmt="int8", type="bf16", layers=1, heads=16, kvh=4, dim=64, seqs=32,
             rows_lo=1, rows_hi=4, past_lo=20000, past_hi=60000, causal=True, window=2048, sinks=4),
        # prompts behind a shared history, grouped heads
        dict(name="attend-prompts", op="attend", fmt="e4m3", type="bf16", layers=1, heads=32, kvh=8, dim=128, seqs=4,
             rows_lo=1000, rows_hi=4097, past_lo=0, past_hi=2000, causal=True, window=0, sinks=0),
        # long inputs read with a window, in 32 bits
        dict(name="attend-window", op="attend", fmt="int8", type="f32", layers=1, heads=8, kvh=8, dim=128, seqs=3,
             rows_lo=2000, rows_hi=6001, past_lo=0, past_hi=300, causal=True, window=1024, sinks=16),
        # one beam step of a single utterance: 5 beams continue from 5 parents, each one row longer
        dict(name="beams-one", op="beams", fmt="int8", layers=8, kvh=8, dim=128, groups=1, beams=5, past_lo=100,
             past_hi=100, pages=256),
        # the same for 64 utterances of 8 beams
        dict(name="beams-batch", op="beams", fmt="e4m3", layers=8, kvh=8, dim=128, groups=64, beams=8, past_lo=20,
             past_hi=700, pages=8192),
        # a pool whose live pages lie scattered after many sequences ended, moved to its start
        dict(name="compact", op="compact", fmt="int8", layers=4, kvh=8, dim=128, seqs=256, past_lo=30, past_hi=500,
             pages=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "beams", "compact"])
    c = dict(op=op, fmt=rng.choice(["e4m3", "int8"]), layers=rng.randint(1, 3), kvh=rng.choice([1, 2, 4, 8]),
             dim=rng.choice([64, 128]))
    if op == "append":
        rows = _log(rng, 1, 3000)
        c.update(type=rng.choice(["f32", "bf16"]), seqs=_log(rng, 1, max(1, min(200, 40000 // rows))),
                 rows_lo=max(1, rows // 3), rows_hi=rows, past_lo=0, past_hi=_log(rng, 1, 800))
    elif op == "attend":
        kind = rng.choice(["step", "few", "prompt"])
        rows = 1 if kind == "step" else rng.randint(2, 24) if kind == "few" else _log(rng, 30, 3000)
        group = rng.choice([1, 1, 2, 3, 4, 8])
        past = _log(rng, 8, 30000 if kind != "prompt" else 2000)
        room = 400000 // (past + rows) if kind != "prompt" else 4000 // rows
        causal = rng.random() < 0.8
        windowed = causal and rng.random() < 0.4
        c.update(type=rng.choice(["f32", "bf16"]), heads=c["kvh"] * group, seqs=max(1, min(_log(rng, 1, 64), room)),
                 rows_lo=max(1, rows // 2), rows_hi=rows, past_lo=past // 4, past_hi=past, causal=causal,
                 window=_log(rng, 20, 4000) if windowed else 0, sinks=rng.choice([0, 1, 4, 33]) if windowed else 0)
    elif op == "beams":
        groups, beams, past = _log(rng, 1, 60), rng.randint(2, 8), _log(rng, 5, 600)
        c.update(groups=groups, beams=beams, past_lo=max(1, past // 4), past_hi=past)
        c["pages"] = groups * beams * (past // ROWS + 3) + rng.randint(0, 500)
    else:
        seqs, past = _log(rng, 1, 250), _log(rng, 5, 500)
        c.update(seqs=seqs, past_lo=1, past_hi=past)
        c["pages"] = int(seqs * (past // ROWS + 1) * rng.uniform(1.3, 3.0)) + 5
    return c


def _lens(case, n):
    """Rows of this call and rows before it, for each of n sequences: the case's extremes, then spread between."""
    rng = random.Random(11)
    lo, hi = case.get("rows_lo", 1), case.get("rows_hi", 1)
    rows = [hi if i == 0 else rng.randint(lo, hi) for i in range(n)]
    past = [case["past_hi"] if i == 0 else rng.randint(case["past_lo"], case["past_hi"]) for i in range(n)]
    return rows, past


def _pages_of(n):
    return (n + ROWS - 1) // ROWS


# ---- inputs --------------------------------------------------------------------------------------------------------
def _scale_of(amax, fmt):
    """The smallest power of two that brings amax within the codes' range (2^-126 for a block of zeros)."""
    top, shift = (448.0, 8) if fmt == "e4m3" else (127.0, 6)
    m, e = torch.frexp(amax)                                       # amax = m 2^e, m in [0.5, 1)
    e = e - 1 - shift + (2 * m > top / 2.0 ** shift).to(e.dtype)
    s = torch.ldexp(torch.ones_like(amax), e.clamp(-126, 120))
    return torch.where(amax > 0, s, torch.full_like(s, 2.0 ** -126))


def _encode(x, scale, fmt):
    y = x * torch.reciprocal(scale)                                # a power of two: exact
    if fmt == "e4m3":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)


def _decode(codes, fmt):
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _values(codes, fmt):
    return codes.view(torch.float8_e4m3fn) if fmt == "e4m3" else codes.view(torch.int8)


def _fill(codes, scales, fmt, gen):
    """Pages of rows as projections give them: normal, a few wide channels, heads of different size."""
    P, L, _, H, R, D = codes.shape
    wide = 1.0 + 3.0 * (torch.rand(L, 2, H, 1, D, device="cuda", generator=gen) > 0.97)
    size = torch.exp(0.5 * torch.randn(L, 2, H, 1, 1, device="cuda", generator=gen))
    step = max(1, (1 << 26) // (L * 2 * H * R * D))
    for p in range(0, P, step):
        n = min(step, P - p)
        x = torch.randn(n, L, 2, H, R, D, device="cuda", generator=gen) * wide * size
        s = _scale_of(x.abs().amax((-2, -1)), fmt)
        scales[p:p + n] = s
        codes[p:p + n] = _encode(x, s[..., None, None], fmt)


def _cache(case, pages, gen):
    shape = (pages, case["layers"], 2, case["kvh"])
    codes = torch.empty(*shape, ROWS, case["dim"], dtype=torch.uint8, device="cuda")
    scales = torch.empty(*shape, device="cuda")
    _fill(codes, scales, case["fmt"], gen)
    return dict(codes=codes, scales=scales, refs=torch.zeros(pages, dtype=torch.int32, device="cuda"))


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _rows(n, heads, dim, gen, kind, size=1.0):
    x = torch.randn(n, heads, dim, device="cuda", generator=gen) * size
    return x if kind == "f32" else x.to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    st = dict(case=case)
    if case["op"] in ("append", "attend"):
        rows, past = _lens(case, case["seqs"])
        lens = [a + b for a, b in zip(rows, past)]
        need = [_pages_of(n) for n in lens]
        total = sum(need)
        width = max(need)
        order = list(range(total + 3))
        rng.shuffle(order)
        table, at = [], 0
        for n in need:
            table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        st.update(_cache(case, total + 3, gen), table=_dev(table), lens=_dev(lens), rows=rows, past=past)
        st["refs"][_dev(order[:total], torch.int64)] = 1
        start = [0]
        for n in rows:
            start.append(start[-1] + n)
        st.update(start=None if max(rows) == 1 else _dev(start), n_rows=start[-1], max_rows=max(rows),
                  max_len=max(lens), layer=case["layers"] - 1)
        if case["op"] == "append":
            st["k"] = _rows(start[-1], case["kvh"], case["dim"], gen, case["type"], 1.5)
            st["v"] = _rows(start[-1], case["kvh"], case["dim"], gen, case["type"], 0.7)
        else:
            st["q"] = _rows(start[-1], case["heads"], case["dim"], gen, case["type"])
    elif case["op"] == "beams":
        n = case["groups"] * case["beams"]
        _, past = _lens(case, case["groups"])
        width = _pages_of(case["past_hi"]) + 2
        order = list(range(case["pages"]))
        rng.shuffle(order)
        table, lens, parents, refs, at = [], [], [], [0] * case["pages"], 0
        for g in range(case["groups"]):
            # beams of one utterance share their full pages but the last, and have a tail of their own
            full, tail = past[g] // ROWS, past[g] % ROWS
            shared = order[at:at + max(0, full - 1)]
            at += len(shared)
            for b in range(case["beams"]):
                mine = order[at:at + (min(full, 1) + (tail > 0))]
                at += len(mine)
                row = shared + mine
                for p in row:
                    refs[p] += 1
                table.append(row + [-1] * (width - len(row)))
                lens.append(past[g])
                parents.append(g * case["beams"] + rng.randint(0, case["beams"] - 1))
        st.update(_cache(case, case["pages"], gen), table=_dev(table), lens=_dev(lens), parents=_dev(parents),
                  new_table=torch.full((n, width), -1, dtype=torch.int32, device="cuda"),
                  new_lens=torch.zeros(n, dtype=torch.int32, device="cuda"), add=_dev([1] * n))
        st["refs"].copy_(_dev(refs))
    else:
        _, lens = _lens(case, case["seqs"])
        width = _pages_of(max(lens))
        order = list(range(case["pages"]))
        rng.shuffle(order)
        table, refs, at = [], [0] * case["pages"], 0
        for s, n in enumerate(lens):
            need = _pages_of(n)
            share = min(need, _pages_of(lens[s - 1])) // 2 if s % 4 == 3 else 0    # a fork of the one before
            row = (table[s - 1][:share] if share else []) + order[at:at + need - share]
            at += need - share
            for p in row:
                refs[p] += 1
            table.append(row + [-1] * (width - need))
        st.update(_cache(case, case["pages"], gen), table=_dev(table), lens=_dev(lens),
                  new_table=torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"),
                  new_refs=torch.zeros(case["pages"], dtype=torch.int32, device="cuda"),
                  live=torch.zeros(1, dtype=torch.int32, device="cuda"))
        st["refs"].copy_(_dev(refs))
    if own:
        kv8 = importlib.import_module("cohere-transcribe_b200.kv8")
        st["cache"] = kv8.Cache(st["codes"], st["scales"], st["refs"], case["fmt"])
        st["seqs"] = kv8.Seqs(st["table"], st["lens"])
        if case["op"] == "beams":
            st["new_seqs"] = kv8.Seqs(st["new_table"], st["new_lens"])
            st["ws"] = st["cache"].pages_workspace(st["new_seqs"])
        elif case["op"] == "compact":
            st["ws"] = st["cache"].pages_workspace(st["seqs"])
        elif case["op"] == "attend":
            st["ws"] = st["cache"].attend_workspace(st["seqs"], st["q"], max_rows=st["max_rows"],
                                                    max_len=st["max_len"], causal=case["causal"],
                                                    window=case["window"], sinks=case["sinks"])
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _plain_append(st):
    """All touched blocks of all sequences side by side: [sequences, blocks, 16 rows, heads, dim]."""
    case = st["case"]
    fmt, layer = case["fmt"], st["layer"]
    S, R = st["lens"].numel(), st["max_rows"]
    ends = st["lens"].long()
    start = st["start"].long() if st["start"] is not None else torch.arange(S + 1, device="cuda")
    past = ends - (start[1:] - start[:-1])
    first = past // ROWS
    blk = first[:, None] + torch.arange((R + ROWS - 2) // ROWS + 1, device="cuda")
    valid = blk * ROWS < ends[:, None]
    tok = blk[..., None] * ROWS + torch.arange(ROWS, device="cuda")
    new = (tok >= past[:, None, None]) & (tok < ends[:, None, None])
    there = (tok < past[:, None, None])[valid]
    row = (start[:-1] - past)[:, None, None] + tok
    page = torch.gather(st["table"].long(), 1, blk.clamp(max=st["table"].shape[1] - 1))[valid]
    pick = new[valid]
    row = torch.where(pick, row[valid], torch.zeros_like(row[valid]))
    for kv, src in ((0, st["k"]), (1, st["v"])):
        x = (src[row].float() * pick[..., None, None]).transpose(1, 2)           # [blocks, heads, 16, dim]
        codes, before = st["codes"][page, layer, kv], st["scales"][page, layer, kv]
        scale = _scale_of(x.abs().amax((-2, -1)), fmt)
        scale = torch.where(there.any(-1)[:, None], torch.maximum(scale, before), scale)
        again = _encode(_decode(codes, fmt), (scale / before)[..., None, None], fmt)
        codes = torch.where(there[:, None, :, None], again, codes)
        codes = torch.where(pick[:, None, :, None], _encode(x, scale[..., None, None], fmt), codes)
        st["codes"][page, layer, kv] = codes
        st["scales"][page, layer, kv] = scale
    return [_values(st["codes"], fmt), st["scales"]]


def _softmax_sum(q, K, V, see):
    """q [..., rows, dim], K and V [..., keys, dim]; rows see at least one key."""
    x = (q @ K.transpose(-1, -2)) * q.shape[-1] ** -0.5
    if see is not None:
        x.masked_fill_(~see, NONE)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (p @ V) / p.sum(-1, keepdim=True)


def _sees(case, at, key, end):
    """Whether the row at token row `at` sees `key`, of a sequence of `end` rows."""
    see = key < end
    if case["causal"]:
        see = see & (key <= at)
        if case["window"]:
            see = see & ((key > at - case["window"]) | (key < case["sinks"]))
    return see


def _plain_attend(st):
    case = st["case"]
    H, Hk, D, S, R = case["heads"], case["kvh"], case["dim"], st["lens"].numel(), st["max_rows"]
    G, fmt, layer = H // Hk, case["fmt"], st["layer"]
    if S * H * R * st["max_len"] <= 1 << 27 and S * st["max_len"] * Hk * D <= 1 << 28:
        # short ones: every sequence padded to the longest
        ends = st["lens"].long()
        start = st["start"].long() if st["start"] is not None else torch.arange(S + 1, device="cuda")
        n = start[1:] - start[:-1]
        i = torch.arange(R, device="cuda")
        row = (start[:-1, None] + i).clamp(max=st["n_rows"] - 1)
        q = st["q"][row].float().view(S, R, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hk, G * R, D)
        kv = _decode(st["codes"][st["table"].clamp_min(0).long(), layer], fmt)
        kv = kv * st["scales"][st["table"].clamp_min(0).long(), layer][..., None, None]
        kv = kv.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)                           # [2, S, heads, keys, dim]
        key = torch.arange(kv.shape[3], device="cuda")
        kv = kv * (key < ends[:, None])[None, :, None, :, None]
        see = _sees(case, ((ends - n)[:, None] + i)[..., None], key, ends[:, None, None])[:, None, None]
        see = see.expand(S, Hk, G, R, key.numel()).reshape(S, Hk, G * R, key.numel())
        o = _softmax_sum(q, kv[0], kv[1], see).view(S, Hk, G, R, D).permute(0, 3, 1, 2, 4).reshape(S, R, H, D)
        return [o[i < n[:, None]].to(st["q"].dtype)]
    out = torch.empty_like(st["q"])
    r0 = 0
    for s, (n, past) in enumerate(zip(st["rows"], st["past"])):
        end = past + n
        lo = max(0, past - case["window"] + 1) // ROWS if case["window"] else 0  # pages that any row sees
        blocks = list(range(min(lo, _pages_of(case["sinks"])))) + list(range(lo, _pages_of(end)))
        blocks = torch.tensor(blocks, device="cuda")
        key = (blocks[:, None] * ROWS + torch.arange(ROWS, device="cuda")).flatten()
        pages = st["table"][s].long()[blocks]
        kv = _decode(st["codes"][pages, layer], fmt) * st["scales"][pages, layer][..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4).flatten(2, 3)                              # [2, heads, keys, dim]
        kv = kv * (key < end)[:, None]
        step = max(1, (1 << 28) // (H * key.numel()))
        for a in range(0, n, step):
            b = min(n, a + step)
            q = st["q"][r0 + a:r0 + b].float().view(b - a, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * (b - a), D)
            see = _sees(case, torch.arange(past + a, past + b, device="cuda")[:, None], key, end)
            see = see.expand(b - a, key.numel()).repeat(G, 1)
            o = _softmax_sum(q, kv[0], kv[1], see)
            out[r0 + a:r0 + b] = o.view(Hk, G, b - a, D).permute(2, 0, 1, 3).reshape(b - a, H, D)
        r0 += n
    return [out]


def _plain_beams(st):
    """Each beam takes its parent's row: full pages are shared, a started page is copied to the lowest free page;
    then every beam gets room for one row more, and the new beams are dropped again."""
    table, lens, refs = st["table"], st["lens"].long()[st["parents"].long()], st["refs"]
    n, width = st["new_table"].shape
    held = (lens + ROWS - 1) // ROWS
    j = torch.arange(width, device="cuda")
    rows = table[st["parents"].long()]
    st["new_table"].copy_(torch.where(j < held[:, None], rows, st["new_table"]))
    tail = lens % ROWS > 0
    shared = j < (lens // ROWS)[:, None]
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    who = torch.nonzero(tail)[:, 0]
    fresh = torch.nonzero(refs == 0)[:who.numel(), 0]
    last = held[who] - 1
    st["codes"][fresh] = st["codes"][rows[who, last].long()]
    st["scales"][fresh] = st["scales"][rows[who, last].long()]
    st["new_table"][who, last] = fresh.int()
    refs[fresh] = 1
    more = torch.nonzero(lens % ROWS == 0)[:, 0]                    # a row more starts a page
    fresh = torch.nonzero(refs == 0)[:more.numel(), 0]
    st["new_table"][more, held[more]] = fresh.int()
    refs[fresh] = 1
    now = (lens + 1 + ROWS - 1) // ROWS
    mine = st["new_table"][j < now[:, None]].long()
    refs.index_add_(0, mine, torch.full_like(mine, -1, dtype=torch.int32))
    st["new_lens"].zero_()
    return [st["new_table"], st["new_lens"], refs, _values(st["codes"], st["case"]["fmt"]), st["scales"]]


def _plain_compact(st):
    """Live pages above the number of live pages move, in order, to the free pages below it."""
    refs = st["refs"]
    P = refs.numel()
    live = refs > 0
    L = live.sum()
    page = torch.arange(P, device="cuda")
    src, dst = torch.nonzero(live & (page >= L))[:, 0], torch.nonzero(~live & (page < L))[:, 0]
    st["codes"][dst] = st["codes"][src]
    st["scales"][dst] = st["scales"][src]
    to = page.int()
    to[src] = dst.int()
    st["new_refs"].zero_()
    st["new_refs"][to[live].long()] = refs[live]
    held = (st["lens"] + ROWS - 1) // ROWS
    used = torch.arange(st["table"].shape[1], device="cuda") < held[:, None]
    st["new_table"].copy_(torch.where(used, to[st["table"].clamp_min(0).long()], st["new_table"]))
    st["live"].copy_(L)
    return [st["new_table"], st["new_refs"], st["live"], _values(st["codes"], st["case"]["fmt"]), st["scales"]]


# ---- the framework's ---------------------------------------------------------------------------------------------
def _own(st):
    case, cache = st["case"], st["cache"]
    if case["op"] == "append":
        cache.append(st["layer"], st["seqs"], st["k"], st["v"], row_start=st["start"], max_rows=st["max_rows"])
        return [_values(st["codes"], case["fmt"]), st["scales"]]
    if case["op"] == "attend":
        return [cache.attend(st["layer"], st["seqs"], st["q"], row_start=st["start"], max_rows=st["max_rows"],
                             max_len=st["max_len"], causal=case["causal"], window=case["window"],
                             sinks=case["sinks"], ws=st["ws"])]
    if case["op"] == "beams":
        cache.fork(st["seqs"], st["parents"], st["new_seqs"], ws=st["ws"])
        cache.reserve(st["new_seqs"], st["add"], ws=st["ws"])
        cache.free(st["new_seqs"])
        return [st["new_table"], st["new_lens"], st["refs"], _values(st["codes"], case["fmt"]), st["scales"]]
    cache.compact(st["seqs"], st["new_refs"], st["new_table"], n_live=st["live"], ws=st["ws"])
    return [st["new_table"], st["new_refs"], st["live"], _values(st["codes"], case["fmt"]), st["scales"]]


def run(st):
    if own:
        return _own(st)
    return {"append": _plain_append, "attend": _plain_attend, "beams": _plain_beams,
            "compact": _plain_compact}[st["case"]["op"]](st)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def _seen(n, past, case):
    """Pairs of a query row and a key that it sees, and keys that any row sees."""
    if not case["causal"]:
        return n * (past + n), past + n
    w, k = case["window"], case["sinks"]
    if not w:
        return n * past + n * (n + 1) // 2, past + n
    pairs = 0
    for i in range(past, past + n):
        lo = max(0, i - w + 1)
        pairs += i + 1 - lo + min(k, lo)
    lo = max(0, past - w + 1)
    return pairs, past + n - lo + min(k, lo)


def work(case):
    D, Hk = case["dim"], case["kvh"]
    if case["op"] in ("append", "attend"):
        size = 4 if case["type"] == "f32" else 2
        rows, past = _lens(case, case["seqs"])
        if case["op"] == "append":
            blocks = sum(_pages_of(a + b) - b // ROWS for a, b in zip(rows, past))
            return dict(bytes=2 * Hk * (sum(rows) * D * (size + 1) + blocks * 4), flops=2 * 2 * Hk * sum(rows) * D)
        seen = [_seen(a, b, case) for a, b in zip(rows, past)]
        keys = sum(k for _, k in seen)
        return dict(bytes=2 * keys * Hk * D + 2 * _pages_of(keys) * Hk * 4 + 2 * sum(rows) * case["heads"] * D * size,
                    flops=4 * D * case["heads"] * sum(p for p, _ in seen))
    page = case["layers"] * 2 * Hk * (ROWS * D + 4)
    if case["op"] == "beams":
        _, past = _lens(case, case["groups"])
        copied = sum(case["beams"] for n in past if n % ROWS)
        entries = sum(case["beams"] * _pages_of(n) for n in past)
        return dict(bytes=2 * copied * page + entries * (8 + 16), flops=0)
    _, lens = _lens(case, case["seqs"])
    need = [_pages_of(n) for n in lens]
    own_pages = sum(n - (min(n, need[s - 1]) // 2 if s % 4 == 3 else 0) for s, n in enumerate(need))
    moved = own_pages * (1.0 - own_pages / case["pages"])          # live pages lie anywhere with equal chance
    return dict(bytes=int(2 * moved * page + sum(need) * 8 + case["pages"] * 8), flops=0)


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------
def _nearest_code(y, fmt):
    """Values that the codes stand for, nearest to y (ties to even), |y| within the codes' range."""
    if fmt == "int8":
        return torch.round(y)
    mag = y.abs()
    e = torch.floor(torch.log2(mag.clamp_min(2.0 ** -6)))
    e = e + (torch.exp2(e + 1) <= mag).to(e.dtype) - (torch.exp2(e) > mag.clamp_min(2.0 ** -6)).to(e.dtype)
    step = torch.exp2(e.clamp_min(-6.0) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    fmt = case["fmt"]
    if case["op"] == "append":
        top = 448.0 if fmt == "e4m3" else 127.0
        D = case["dim"]
        codes, scales = _values(st["codes"], fmt).double(), st["scales"].double()
        table = st["table"].tolist()
        r0 = 0
        for s, (n, past) in enumerate(zip(st["rows"], st["past"])):
            for b in range(past // ROWS, _pages_of(past + n)):
                page, lo, hi = table[s][b], max(past, b * ROWS), min(past + n, (b + 1) * ROWS)
                there = lo - b * ROWS
                x = torch.stack([t[r0 + lo - past:r0 + hi - past].double().transpose(0, 1) for t in
                                 (st["k"], st["v"])])               # [2, heads, rows, dim]
                amax = x.abs().amax((-2, -1))
                e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -150) / top))
                e = e - (torch.exp2(e - 1) * top >= amax).double() + (torch.exp2(e) * top < amax).double()
                sc = torch.exp2(e.clamp_min(-126.0))
                if there:
                    before = scales[page, st["layer"]]
                    sc = torch.maximum(sc, before)
                    old = codes[page, st["layer"], :, :, :there]
                    codes[page, st["layer"], :, :, :there] = _nearest_code(old * (before / sc)[..., None, None], fmt)
                codes[page, st["layer"], :, :, there:hi - b * ROWS] = _nearest_code(x / sc[..., None, None], fmt)
                scales[page, st["layer"]] = sc
            r0 += n
        return [codes, scales]
    if case["op"] == "attend":
        if work(case)["flops"] > 2e12:
            return None
        H, Hk, D = case["heads"], case["kvh"], case["dim"]
        G = H // Hk
        out = torch.empty(st["n_rows"], H, D, dtype=torch.float64, device="cuda")
        r0 = 0
        for s, (n, past) in enumerate(zip(st["rows"], st["past"])):
            L = past + n
            pages = st["table"][s, :_pages_of(L)].long()
            for h in range(Hk):
                blk = _decode(st["codes"][pages, st["layer"], :, h], fmt).double()
                blk = blk * st["scales"][pages, st["layer"], :, h].double()[..., None, None]
                K, V = (blk[:, i].reshape(-1, D)[:L] for i in (0, 1))
                for a in range(0, n, 1024):
                    b = min(n, a + 1024)
                    pos = torch.arange(past + a, past + b, device="cuda").unsqueeze(1)
                    key = torch.arange(L, device="cuda").unsqueeze(0)
                    hide = torch.zeros(b - a, L, dtype=torch.bool, device="cuda")
                    if case["causal"]:
                        hide = key > pos
                        if case["window"]:
                            hide = hide | ((pos - key >= case["window"]) & (key >= case["sinks"]))
                    for g in range(G):
                        x = st["q"][r0 + a:r0 + b, h * G + g].double() @ K.T / math.sqrt(D)
                        out[r0 + a:r0 + b, h * G + g] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ V
            r0 += n
        return [out]
    codes, scales = _values(st["codes"], fmt), st["scales"]
    table, refs = st["table"].tolist(), st["refs"].tolist()
    lens = st["lens"].tolist()
    if case["op"] == "beams":
        new = [[-1] * len(r) for r in table]
        src, dst, grown = [], [], []
        free = iter([p for p, r in enumerate(refs) if r == 0])
        for i, par in enumerate(st["parents"].tolist()):
            for b in range(_pages_of(lens[par])):
                new[i][b] = table[par][b]
                if (b + 1) * ROWS > lens[par]:
                    new[i][b] = next(free)
                    src.append(table[par][b])
                    dst.append(new[i][b])
        for i, par in enumerate(st["parents"].tolist()):
            if lens[par] % ROWS == 0:
                new[i][lens[par] // ROWS] = next(free)
        a, b = _dev(src, torch.int64), _dev(dst, torch.int64)
        codes.view(torch.uint8)[b] = codes.view(torch.uint8)[a]
        scales[b] = scales[a]
        return [_dev(new), torch.zeros(len(new), dtype=torch.int32, device="cuda"), _dev(refs), codes, scales]
    live = [p for p, r in enumerate(refs) if r > 0]
    gaps = [p for p in range(len(live)) if refs[p] == 0]
    move = dict(zip([p for p in live if p >= len(live)], gaps))
    if move:
        a, b = _dev(list(move), torch.int64), _dev(list(move.values()), torch.int64)
        codes.view(torch.uint8)[b] = codes.view(torch.uint8)[a]
        scales[b] = scales[a]
    count = [0] * len(refs)
    for p in live:
        count[move.get(p, p)] = refs[p]
    new = [[move.get(p, p) if b < _pages_of(n) else -1 for b, p in enumerate(r)] for r, n in zip(table, lens)]
    return [_dev(new), _dev(count), _dev([len(live)]), codes, scales]
