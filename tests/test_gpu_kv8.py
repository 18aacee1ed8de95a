"""GPU tests of the 8-bit paged K/V cache (include/ct_kv8.h through kv8.py) against kv8_ref.py's 64-bit loops.

Written codes, scales and everything about pages have to be equal bit for bit: scales are powers of two, so a
value divided by one is exact and its rounding has one answer.

Attention tolerances, derived per output from the kernels' arithmetic.  With reach = scale max|q| max_j sum_d |k_jd|
(an upper bound of any |score|) and mass = sum_j p_j |v_j|:
  a score is off by at most reach * (2^-22 for the query held as two fp16 + (D / 16 + 9) 2^-22 for that many fp32
  steps) + 2^-20 for the exponential, so a probability is off by twice that, relative;
  probabilities as two fp16 add 2^-22, the sums over n pages (n + 64) 2^-22 (in calls of many bf16 rows the
  probability is one fp16: 2^-11 instead);
  an fp16 has an absolute step below its normal numbers: a probability's error is at least 2^-32 of the row's largest
  (2^-28 as one fp16), whatever its own size, which adds that times the sum of |v|;
  all the rest of it scales with mass; rounding the result to its type adds half a step, |out| eps / 2.
"""
import importlib
import math

import numpy as np
import pytest

import kv8_ref as ref

pytestmark = pytest.mark.gpu
BAD_ARG, NO_PAGE = 4, 6
ROWS = ref.ROWS


@pytest.fixture(scope="module")
def kv8():
    return importlib.import_module("cohere-transcribe_b200.kv8")


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def to_values(codes, fmt):
    import torch
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float().cpu().numpy().astype(np.float64)


def random_codes(shape, fmt, gen):
    import torch
    r = torch.randint(0, 256, shape, dtype=torch.int32, device="cuda", generator=gen)
    if fmt == "e4m3":                       # any code but the two NaNs, small exponents as rare as large ones
        r = torch.where((r & 127) == 127, r - 1, r)
    else:
        r = torch.where(r == 128, r + 1, r)
    return r.to(torch.uint8)


def gauss_codes(shape, fmt, gen):
    import torch
    x = torch.randn(shape, device="cuda", generator=gen)
    if fmt == "e4m3":
        return (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return (x * 32).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)


def make(kv8, fmt, lens, kvh, dim, layers=2, spare=5, seed=0, gauss=True, refs=True):
    """A cache whose sequences lie over shuffled pages; scales are powers of two of several sizes."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [ref.pages_of(max(n, 0)) for n in lens]
    pages, width = sum(need) + spare, max(max(need), 1)
    shape = (pages, layers, 2, kvh)
    codes = (gauss_codes if gauss else random_codes)(shape + (ROWS, dim), fmt, gen)
    e = torch.randint(-9, -5, shape, device="cuda", generator=gen)
    scales = torch.ldexp(torch.ones(shape, device="cuda"), e) * (1 if fmt == "int8" else 0.5)
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    r = torch.zeros(pages, dtype=torch.int32, device="cuda")
    for p in order[:at]:
        r[p] = 1
    c = kv8.Cache(codes, scales, r if refs else None, fmt)
    s = kv8.Seqs(torch.tensor(table, dtype=torch.int32, device="cuda"),
                 torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return c, s, ref.Cache(to_values(codes, fmt), scales.cpu().numpy().astype(np.float64), r.cpu().numpy(), fmt), table


def starts_of(rows):
    return [0] + np.cumsum(rows).tolist()


def dev(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same_cache(c, rc):
    assert np.array_equal(to_values(c.codes, c.fmt), rc.v)
    assert np.array_equal(c.scales.cpu().numpy().astype(np.float64), rc.s, equal_nan=True)


# ---- append --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("kvh,dim", [(1, 64), (3, 128)])
@pytest.mark.parametrize("rows,past", [
    ([1, 1, 1, 1], [0, 15, 16, 40]),            # decode rows: a new page, the last row of one, the first
    ([17, 1, 0, 33, 16, 5], [0, 3, 20, 31, 16, 11]),
    ([200, 64], [7, 0]),
])
def test_append_matches_the_definition(kv8, torch, fmt, typ, kvh, dim, rows, past):
    lens = [a + b for a, b in zip(rows, past)]
    c, s, rc, table = make(kv8, fmt, lens, kvh, dim, gauss=False, seed=dim + len(rows))
    gen = torch.Generator(device="cuda").manual_seed(3)
    n = sum(rows)
    # one packed tensor as a projection gives it: q | k | v side by side, rows of different sizes
    qkv = torch.randn(n + 2, 3 * kvh, dim, device="cuda", generator=gen) * torch.exp(
        3 * torch.randn(n + 2, 1, 1, device="cuda", generator=gen))
    qkv = qkv.to(getattr(torch, typ))
    k, v = qkv[1:n + 1, kvh:2 * kvh], qkv[1:n + 1, 2 * kvh:]
    st = starts_of(rows)
    one = max(rows) == 1
    c.append(1, s, k, v, row_start=None if one else dev(st), max_rows=max(rows))
    assert c.status() == 0
    rc.append(1, table, lens, k.float().cpu().numpy(), v.float().cpu().numpy(), st)
    same_cache(c, rc)
    c.append(1, s, k, v, row_start=None if one else dev(st), max_rows=max(rows))   # the same rows again: the same codes
    same_cache(c, rc)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_scales_at_the_borders(kv8, torch, fmt):
    """Rows whose largest magnitude is a border of the codes' range, zeros, subnormals, the largest floats."""
    top = 448.0 if fmt == "e4m3" else 127.0
    c, s, rc, table = make(kv8, fmt, [1] * 10, 1, 64)
    x = torch.zeros(10, 1, 64, device="cuda")
    for i, a in enumerate([0.0, top, np.nextafter(np.float32(top), np.float32(1e9)), top / 2, 1e-38, 1e-45, 3e38,
                           2.0 ** -126, 1.0, float(np.finfo(np.float32).max)]):
        x[i, 0, ::7] = float(a)
        x[i, 0, 1::7] = -float(a) / 3
    c.append(0, s, x, -x)
    assert c.status() == 0
    xs = x.cpu().numpy()
    rc.append(0, table, [1] * 10, xs, -xs, list(range(11)))
    same_cache(c, rc)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_nonfinite_values(kv8, torch, fmt):
    """Infinities saturate, a NaN marks its block (and only it) until the page is begun anew."""
    lens = [20, 20, 33]
    c, s, rc, table = make(kv8, fmt, lens, 2, 64)
    x = torch.randn(33, 2, 64, device="cuda")
    x[2, 0, 5] = float("inf")
    x[3, 1, 6] = -float("inf")
    x[7, 0, 7] = float("nan")
    x[30, 1, 0] = float("nan")
    st = starts_of([5, 5, 23])
    c.append(0, s, x, x.flip(0).contiguous(), row_start=dev(st), max_rows=23)
    xs = x.cpu().numpy()
    rc.append(0, table, lens, xs, xs[::-1], st)
    same_cache(c, rc)
    assert np.isnan(rc.s[:, 0]).sum() == 4
    c.append(0, s, x[10:13], x[10:13])           # one more row: marked blocks stay marked
    rc.append(0, table, lens, xs[10:13], xs[10:13], [0, 1, 2, 3])
    same_cache(c, rc)
    s2 = kv8.Seqs(s.table, dev([1, 1, 1]))       # begun anew
    c.append(0, s2, x[10:13], x[10:13])
    rc.append(0, table, [1, 1, 1], xs[10:13], xs[10:13], [0, 1, 2, 3])
    same_cache(c, rc)
    assert not np.isnan(c.scales[s.table[:, 0].long(), 0].cpu().numpy()).any()


def test_append_leaves_out_what_it_cannot_write(kv8, torch):
    lens = [20, 20, 20, 20, 0]
    c, s, rc, table = make(kv8, "int8", lens, 1, 64)
    before, sc = c.codes.clone(), c.scales.clone()
    s.table[0, 1] = c.n_pages                    # outside the pool
    s.table[1, 1] = -1
    c.refs[table[2][1]] = 2                      # a page that another sequence holds as well
    s.lens[3] = 10 ** 6                          # longer than the table
    x = torch.randn(5, 1, 64, device="cuda")
    c.append(0, s, x, x)                         # row 4: a sequence of length 0 has no row
    assert c.status() == BAD_ARG and c.status() == 0
    assert torch.equal(c.codes, before) and torch.equal(c.scales, sc)
    s.lens[:] = dev([0, 0, 0, 0, 0])
    c.append(0, s, x, x)
    assert c.status() == 0 and torch.equal(c.codes, before)


# ---- attention -----------------------------------------------------------------------------------------------------
def tolerance(out, mass, reach, total, dim, pages, typ, single):
    import torch
    dx = reach * (dim / 16 + 10) * 2.0 ** -22 + 2.0 ** -20
    rel = 2.2 * dx + (2.0 ** -11 if single else 2.0 ** -22) + (pages + 64) * 2.0 ** -22
    return mass * rel + total * 2.0 ** (-28 if single else -32) + np.abs(out) * (torch.finfo(getattr(torch, typ)).eps / 2) + 1e-30


def check_attend(kv8, c, s, rc, table, lens, rows, heads, typ, seed=1, causal=True, window=0, sinks=0, scale=None,
                 layer=1, spread=1.0, max_len=None, pad_rows=3):
    import torch
    D = c.head_dim
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, one = sum(rows), all(r == 1 for r in rows)
    qkv = (torch.randn(n + pad_rows, heads + 1, D, device="cuda", generator=gen) * spread).to(getattr(torch, typ))
    q = qkv[:, 1:]                               # a strided view
    out = torch.full((n + pad_rows, heads, D), 7.0, device="cuda", dtype=q.dtype)
    st = starts_of(rows)
    scale = D ** -0.5 if scale is None else scale
    kw = dict(row_start=None if one else dev(st), max_rows=max(max(rows), 1), causal=causal, window=window,
              sinks=sinks, scale=scale, max_len=max_len)
    got = c.attend(layer, s, q, out=out, **kw)
    assert got is out and c.status() == 0
    assert bool((out[n:] == 7.0).all())          # rows behind the last sequence
    want, mass, reach, total = ref.attend(rc, layer, table, lens, q[:n].float().cpu().numpy(), st, c.kv_heads, scale, causal,
                                   window, sinks)
    o = out[:n].float().cpu().numpy().astype(np.float64)
    tol = tolerance(want, mass, reach, total, D, max(len(r) for r in table), typ, typ == "bfloat16")
    bad = ~(np.abs(o - want) <= tol)
    bad &= ~(np.isnan(o) & np.isnan(want))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(np.abs(o - want) / tol)))
    again = torch.full_like(out, 7.0)
    c.attend(layer, s, q, out=again, **kw)
    assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(out))    # the same bits each time
    return out


SHAPES = [  # kv heads, heads, dim
    (2, 2, 128), (1, 8, 64), (3, 9, 128), (2, 32, 64)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("kvh,heads,dim", SHAPES)
def test_attention_single_rows(kv8, fmt, typ, kvh, heads, dim):
    lens = [1, 2, 16, 17, 100, 333, 64, 0, 1025]
    c, s, rc, table = make(kv8, fmt, lens, kvh, dim, seed=heads)
    check_attend(kv8, c, s, rc, table, lens, [1] * len(lens), heads, typ)
    check_attend(kv8, c, s, rc, table, lens, [1] * len(lens), heads, typ, causal=False, spread=4.0)
    check_attend(kv8, c, s, rc, table, lens, [1] * len(lens), heads, typ, window=40, sinks=5)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("kvh,heads,dim", SHAPES)
@pytest.mark.parametrize("rows,past", [
    ([3, 1, 8, 0, 5], [0, 50, 200, 10, 31]),
    ([40, 17, 33], [0, 100, 15]),
    ([130, 1, 257, 64], [0, 300, 5, 64]),
])
def test_attention_many_rows(kv8, fmt, typ, kvh, heads, dim, rows, past):
    lens = [a + b for a, b in zip(rows, past)]
    c, s, rc, table = make(kv8, fmt, lens, kvh, dim, seed=heads + dim)
    check_attend(kv8, c, s, rc, table, lens, rows, heads, typ)
    check_attend(kv8, c, s, rc, table, lens, rows, heads, typ, causal=False)
    check_attend(kv8, c, s, rc, table, lens, rows, heads, typ, window=23, sinks=18)
    check_attend(kv8, c, s, rc, table, lens, rows, heads, typ, window=1, sinks=0)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_many_rows_over_many_key_tiles(kv8, typ, dim):
    """Pieces of many key tiles: every tile's scores take the place of the tile's probabilities before it."""
    rows, past = [300, 40, 130, 7], [3700, 2461, 0, 900]
    lens = [a + b for a, b in zip(rows, past)]
    c, s, rc, table = make(kv8, "e4m3", lens, 4, dim, seed=dim)
    check_attend(kv8, c, s, rc, table, lens, rows, 8, typ)
    check_attend(kv8, c, s, rc, table, lens, rows, 8, typ, window=1500, sinks=40)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_many_sequences_of_some_rows(kv8, fmt, typ, dim):
    """17 to 32 rows per kv head with enough sequences to fill the GPU: a kernel form of its own."""
    rng = np.random.default_rng(dim)
    rows = [6 if i == 3 else int(rng.integers(0, 7)) for i in range(70)]
    lens = [r + int(rng.integers(0, 120)) for r in rows]
    lens[5] = 1500 + rows[5]
    c, s, rc, table = make(kv8, fmt, lens, 2, dim, seed=dim)
    check_attend(kv8, c, s, rc, table, lens, rows, 10, typ)
    check_attend(kv8, c, s, rc, table, lens, rows, 10, typ, window=33, sinks=2)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads", [17, 40, 128, 300])
def test_attention_large_groups(kv8, typ, heads):
    """One row per sequence, many heads on one kv head: odd groups, tiles that end inside a query row."""
    lens = [70, 1, 300]
    c, s, rc, table = make(kv8, "int8", lens, 1, 64, seed=heads)
    check_attend(kv8, c, s, rc, table, lens, [1, 1, 1], heads, typ)
    check_attend(kv8, c, s, rc, table, lens, [1, 1, 1], heads, typ, window=20, sinks=1)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_attention_in_place(kv8, torch, typ, rows):
    """out may be q: the same bits as into another tensor, with and without pieces to join."""
    for n in (40, 400, 3000):
        c, s, rc, table = make(kv8, "e4m3", [n + rows, rows], 2, 128)
        q = torch.randn(2 * rows, 4, 128, device="cuda").to(getattr(torch, typ))
        st = dev([0, rows, 2 * rows])
        want = c.attend(1, s, q, row_start=st, max_rows=rows)
        c.attend(1, s, q, out=q, row_start=st, max_rows=rows)
        assert torch.equal(q, want)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 6, 300])
def test_attention_window_over_a_long_cache(kv8, typ, rows):
    """Released pages between the sinks and the window are never read; windows end inside pages."""
    lens = [5000, 4097, 300]
    rows = [rows, max(1, rows // 2), 1]
    c, s, rc, table = make(kv8, "int8", lens, 2, 64)
    for i, n in enumerate(lens):
        first = max(0, n - rows[i] - 700) // ROWS
        s.table[i, 3:first] = -1
        for b in range(3, first):
            table[i][b] = -1
    check_attend(kv8, c, s, rc, table, lens, rows, 4, typ, window=700, sinks=37)
    check_attend(kv8, c, s, rc, table, lens, rows, 4, typ, window=512, sinks=0)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 9, 150])
def test_attention_ignores_what_is_hidden(kv8, torch, typ, rows):
    """Codes behind the last row hold NaN patterns, pages that no row sees NaN scales: neither shows."""
    lens = [rows + 70, rows + 3, rows]
    rws = [rows] * 3
    c, s, rc, table = make(kv8, "e4m3", lens, 2, 128)
    for i, n in enumerate(lens):
        t = n % ROWS
        if t:
            p = table[i][n // ROWS]
            c.codes[p, :, :, :, t:] = 0x7F
            rc.v[p, :, :, :, t:] = np.nan
    rc.v = np.nan_to_num(rc.v)
    used = {p for r in table for p in r if p >= 0}
    for p in range(c.n_pages):
        if p not in used:
            c.scales[p] = float("nan")
    check_attend(kv8, c, s, rc, table, lens, rws, 4, typ)
    check_attend(kv8, c, s, rc, table, lens, rws, 4, typ, causal=False)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 12, 200])
@pytest.mark.parametrize("kv", [0, 1])
def test_attention_marked_blocks_reach_only_rows_that_see_them(kv8, typ, rows, kv):
    lens = [rows + 20, rows + 100]
    c, s, rc, table = make(kv8, "int8", lens, 2, 64)
    for i, b in ((0, lens[0] // ROWS), (1, 2)):
        p = table[i][min(b, ref.pages_of(lens[i]) - 1)]
        c.scales[p, 1, kv, 0] = float("nan")
        rc.s[p, 1, kv, 0] = np.nan
    o = check_attend(kv8, c, s, rc, table, lens, [rows] * 2, 4, typ, window=30, sinks=0)
    assert bool(o[:, 2:].isfinite().all())       # the other kv head's rows
    check_attend(kv8, c, s, rc, table, lens, [rows] * 2, 4, typ)


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [[1, 1], [20, 5], [300, 200]])
def test_attention_rows_that_see_nothing(kv8, torch, typ, rows):
    """More rows than the sequence has: the ones before token row 0 get zeros; so does an empty sequence."""
    lens = [rows[0] // 2, 0]
    c, s, rc, table = make(kv8, "int8", lens, 1, 64)
    o = check_attend(kv8, c, s, rc, table, lens, rows, 2, typ)
    assert bool((o[:rows[0] - lens[0]] == 0).all()) and bool((o[rows[0]:sum(rows)] == 0).all())


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 150])
def test_attention_uneven_block_scales(kv8, torch, typ, rows):
    """Block scales over a wide range, zero among them, and scales that are no powers of two."""
    lens = [rows + 200, rows + 40]
    c, s, rc, table = make(kv8, "int8", lens, 2, 128)
    gen = torch.Generator(device="cuda").manual_seed(4)
    f = torch.exp(torch.randn(c.scales.shape, device="cuda", generator=gen))
    f[:, :, 1] *= torch.exp(2 * torch.randn(f[:, :, 1].shape, device="cuda", generator=gen))
    c.scales.mul_(f)
    c.scales[::5, :, 1] = 0
    rc.s = c.scales.cpu().numpy().astype(np.float64)
    check_attend(kv8, c, s, rc, table, lens, [rows] * 2, 6, typ)


def row_bounds(rc, layer, table, lens, q, starts, scale, causal, window, sinks, typ, tiny=1e-37):
    """Attention in 64 bits, and what its rounding errors may add up to when each key's are counted by what the key adds
    (reach, masses and sums as above, but none of them may be excused by a key that a row hardly feels):
      a probability is off by at most dx of its own key, relative: sum_j p_j dx_j (|v_j| + |out|);
      its fp16 form by 2^-22 (one fp16: 2^-11), and the sums by (pages + 64) 2^-22, relative to mass;
      an fp16's absolute step 2^-24, that is 2^-25 an entry, counts in units of which the row's largest product of
      probability and V scale is at least 2^8: 2^-33 max_j(p_j scale_j) sum |code|."""
    import torch
    R, H, D = q.shape
    G, pages = H // rc.v.shape[3], max(len(r) for r in table)
    out, tol = np.zeros((R, H, D)), np.zeros((R, H, D))
    for s, L in enumerate(lens):
        n, rows = starts[s + 1] - starts[s], slice(starts[s], starts[s + 1])
        row = table[s][:ref.pages_of(L)]
        t, j = L - n + np.arange(n)[:, None], np.arange(L)[None]
        see = np.broadcast_to(ref.sees(t, j, L, causal, window, sinks), (n, L))
        for h in range(H):
            K, V = rc.rows(layer, row, L, h // G)
            unit = np.repeat(rc.s[row, layer, 1, h // G], ROWS)[:L]
            code = np.abs(rc.v[row, layer, 1, h // G].reshape(-1, D)[:L])
            x = np.where(see, scale * (q[rows, h] @ K.T), -np.inf)
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            reach = scale * np.abs(q[rows, h]).max(1, keepdims=True) * np.abs(K).sum(1)
            dx = 1.1 * (reach * (D / 16 + 10) * 2.0 ** -22 + 2.0 ** -20)
            o, mass = p @ V, p @ np.abs(V)
            rel = (2.0 ** -11 if typ == "bfloat16" else 2.0 ** -22) + (pages + 64) * 2.0 ** -22
            out[rows, h] = o
            tol[rows, h] = ((p * dx) @ np.abs(V) + (p * dx).sum(1, keepdims=True) * np.abs(o) + mass * rel
                            + 2.0 ** -33 * (p * unit).max(1, keepdims=True) * (see @ code)
                            + np.abs(o) * (torch.finfo(getattr(torch, typ)).eps / 2) + tiny)
    return out, tol


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,heads", [(1, 2), (1, 8), (5, 12), (150, 4)])
@pytest.mark.parametrize("place", ["first", "last", "spread"])
def test_attention_value_scales_far_apart(kv8, torch, fmt, typ, rows, heads, place):
    """Blocks whose V scale is 2^k times the others' and whose probability is 2^-k of theirs, or next to nothing:
    the others keep their bits."""
    dim, kvh, n = 64, 2, 600
    lens, st = [n + rows, 200 + rows], [0, rows, 2 * rows]
    for k in (10, 20, 30, 40):
        for drop in (k, 200):
            c, s, rc, table = make(kv8, fmt, lens, kvh, dim, seed=k + drop)
            gen = torch.Generator(device="cuda").manual_seed(k)
            q = (torch.randn(2 * rows, heads, dim, device="cuda", generator=gen).abs() + 0.5).to(getattr(torch, typ))
            for i, L in enumerate(lens):
                big = {"first": range(0, 9), "last": range(L // ROWS - 4, L // ROWS), "spread": range(1, L // ROWS, 3)}[place]
                for b in big:
                    page = table[i][b]
                    # K rows of -1 times a factor: q's mean entry is about 1.3, so a score falls by 0.125 * 64 * 1.3 of it
                    c.codes[page, 1, 0] = 0xB8 if fmt == "e4m3" else 0xFF              # -1
                    c.scales[page, 1, 0] = drop * math.log(2) / (0.125 * 64 * 1.3)
                    c.scales[page, 1, 1] *= 2.0 ** k
            rc = ref.Cache(to_values(c.codes, fmt), c.scales.cpu().numpy().astype(np.float64), rc.refs, fmt)
            got = c.attend(1, s, q, row_start=dev(st), max_rows=rows).double().cpu().numpy()
            want, tol = row_bounds(rc, 1, table, lens, q.double().cpu().numpy(), st, 0.125, True, 0, 0, typ)
            assert c.status() == 0
            worst = np.abs(got - want) / tol
            assert (worst <= 1).all(), (k, drop, float(np.nanmax(worst)), float(np.abs(got - want).max()))


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,past", [(1, 1), (1, 700), (3, 40), (150, 20), (150, 2000)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_attention_nonfinite_queries(kv8, torch, typ, rows, past, value):
    """A row whose query holds an infinity or a NaN is NaN, as its softmax is, whatever the signs in K; the other rows and
    heads do not feel it, and a row that sees nothing stays zero."""
    lens, st = [past + rows, rows - 1], [0, rows, 2 * rows]
    c, s, rc, table = make(kv8, "int8", lens, 2, 64)
    c.codes[:, 1, 0, 0, :, 3] = 0xFF if value > 0 else 1       # every K of kv head 0 has -1 (or 1) there
    q = torch.randn(2 * rows, 4, 64, device="cuda").to(getattr(torch, typ))
    want = c.attend(1, s, q, row_start=dev(st), max_rows=rows)
    q[0, 1, 3] = q[rows - 1, 0, 3] = q[rows, 1, 3] = value
    got = c.attend(1, s, q, row_start=dev(st), max_rows=rows)
    assert c.status() == 0
    hit = torch.zeros(2 * rows, 4, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[rows - 1, 0] = True
    assert bool(got[hit].isnan().all()) and bool((got[rows] == 0).all())     # row `rows` is before its first token row
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [2e38, 1e37, 1e-36])
@pytest.mark.parametrize("rows,past,heads", [(1, 40, 2), (1, 700, 2), (1, 6000, 8), (3, 3000, 10), (150, 20, 4), (150, 3000, 4)])
def test_attention_of_values_near_the_ends_of_fp32(kv8, torch, typ, size, rows, past, heads):
    """A result lies between the values it is made of: it overflows nowhere on its way, and small ones keep their
    bits. One row and several, one piece, a cluster's pieces and those that a second kernel joins."""
    kvh, dim = 2, 64
    lens, st = [past + rows, past // 2 + rows], [0, rows, 2 * rows]
    c, s, rc, table = make(kv8, "e4m3", lens, kvh, dim)
    gen = torch.Generator(device="cuda").manual_seed(1)
    kv = [torch.rand(sum(lens), kvh, dim, device="cuda", generator=gen) - 0.5 for _ in range(2)]
    c.append(1, s, kv[0], kv[1] * size * 2, row_start=dev(starts_of(lens)), max_rows=max(lens))
    q = torch.randn(2 * rows, heads, dim, device="cuda", generator=gen).to(getattr(torch, typ))
    rc = ref.Cache(to_values(c.codes, "e4m3"), c.scales.cpu().numpy().astype(np.float64), rc.refs, "e4m3")
    got = c.attend(1, s, q, row_start=dev(st), max_rows=rows).double().cpu().numpy()
    # below the smallest normal number, 2^-126, a product's step is 2^-149 (a few of them), and the type's own 2^-126 eps
    tiny = 2.0 ** -146 + 2.0 ** -126 * torch.finfo(getattr(torch, typ)).eps / 2
    want, tol = row_bounds(rc, 1, table, lens, q.double().cpu().numpy(), st, 0.125, True, 0, 0, typ, tiny=tiny)
    assert c.status() == 0 and np.isfinite(want.astype(np.float32)).all()
    worst = np.abs(got - want) / tol
    assert (worst <= 1).all(), (float(np.nanmax(worst)), int((~np.isfinite(got)).sum()))


def test_attention_extreme_queries(kv8, torch):
    """Very large and very small queries, and a scale that makes one key take all."""
    lens = [90, 40]
    c, s, rc, table = make(kv8, "e4m3", lens, 1, 64)
    for spread, scale in ((1e-30, 1e27), (1e20, 1e-23), (1.0, 3.0), (0.0, 1.0)):
        check_attend(kv8, c, s, rc, table, lens, [1, 1], 2, "float32", spread=spread, scale=scale)
        check_attend(kv8, c, s, rc, table, lens, [70, 40], 2, "float32", spread=spread, scale=scale)


def test_attention_leaves_out_bad_sequences(kv8, torch):
    lens = [40, 40, 40]
    c, s, rc, table = make(kv8, "int8", lens, 1, 64)
    q = torch.randn(3, 1, 64, device="cuda")
    good = c.attend(0, s, q)
    s.lens[1] = 49                               # longer than its table row
    out = torch.full_like(q, 7.0)
    c.attend(0, s, q, out=out)
    assert c.status() == BAD_ARG and bool((out[1] == 7).all()) and torch.equal(out[::2], good[::2])
    s.lens[1] = 40
    out = torch.full_like(q, 7.0)
    c.attend(0, s, q, out=out, max_len=39)
    assert c.status() == BAD_ARG and bool((out == 7).all())
    s.table[2, 1] = c.n_pages + 3                # a page outside the pool: its rows count as not there
    got = c.attend(0, s, q)
    assert c.status() == BAD_ARG
    rc1 = ref.Cache(rc.v, rc.s, rc.refs, "int8")
    pages = [table[2][0], table[2][2]]
    want, _, _, _ = ref.attend(rc1, 0, [pages], [24], q[2:].cpu().numpy(), [0, 1], 1, 0.125)
    assert np.allclose(got[2].cpu().numpy(), want[0], rtol=1e-4, atol=1e-5)
    st = dev([0, 1, 50, 3])                      # spans outside the packed rows
    out = torch.full_like(q, 7.0)
    c.attend(0, s, q, out=out, row_start=st, max_rows=50)
    assert c.status() == BAD_ARG and bool((out[1:] == 7).all())


@pytest.mark.parametrize("typ", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 5, 90])
def test_attention_does_not_depend_on_the_other_sequences(kv8, torch, typ, rows):
    lens = [500, 90, 1300]
    c, s, rc, table = make(kv8, "e4m3", lens, 2, 128)
    q = torch.randn(3 * rows, 4, 128, device="cuda").to(getattr(torch, typ))
    st = dev(starts_of([rows] * 3))
    a = c.attend(1, s, q, row_start=st, max_rows=rows)
    c.codes[s.table[0, :32].long()] = 1
    s.lens[2] = 17
    s.table[2, 5:] = -1
    b = c.attend(1, s, q, row_start=st, max_rows=rows)
    if rows <= 17:
        assert c.status() == 0
    assert torch.equal(a[rows:2 * rows], b[rows:2 * rows])


@pytest.mark.parametrize("rows", [1, 4, 100])
def test_attention_on_two_streams(kv8, torch, rows):
    """Two calls over the same cache at once, each with a workspace of its own: the bits of one call alone."""
    c, s, rc, table = make(kv8, "e4m3", [3000 + rows, 700 + rows, rows], 2, 128)
    st = dev(starts_of([rows] * 3))
    qs = [torch.randn(3 * rows, 4, 128, device="cuda") for _ in range(2)]
    want = [c.attend(1, s, q, row_start=st, max_rows=rows) for q in qs]
    ws = [c.attend_workspace(s, q, max_rows=rows) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, w, stream in zip(qs, ws, streams):
            with torch.cuda.stream(stream):
                got.append(c.attend(1, s, q, row_start=st, max_rows=rows, ws=w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert c.status() == 0


@pytest.mark.parametrize("typ,pages_a_piece", [("float32", 1024), ("bfloat16", 4096)])
def test_attention_sums_of_millions_of_keys(kv8, torch, typ, pages_a_piece):
    """33 rows of each of 148 sequences over the same 16.8 million keys: the sums are cut into pieces however long the
    cache. All scores are 0, so a result is the mean of V.  The tensor core truncates each of its sums, one per page of a
    piece, by less than 2^-22 of it; 64 such steps more for the rest, as in the other tests, and half a step of the type."""
    n, seqs, rows = 1 << 20, 148, 33
    gen = torch.Generator(device="cuda").manual_seed(5)
    c = kv8.Cache(torch.zeros(n, 1, 2, 1, ROWS, 64, dtype=torch.uint8, device="cuda"),
                  torch.full((n, 1, 2, 1), 2.0 ** -6, device="cuda"), None, "int8")
    c.codes[:, 0, 1] = torch.randint(60, 128, (n, 1, ROWS, 64), dtype=torch.uint8, device="cuda", generator=gen)
    want = c.codes[:, 0, 1].sum((0, 1, 2), dtype=torch.int64).double() / (n * ROWS * 64)
    s = kv8.Seqs(torch.arange(n, dtype=torch.int32, device="cuda").expand(seqs, n).contiguous(), dev([n * ROWS] * seqs))
    q = torch.randn(seqs * rows, 1, 64, device="cuda", generator=gen).to(getattr(torch, typ))
    out = c.attend(0, s, q, row_start=dev([rows * i for i in range(seqs + 1)]), max_rows=rows, causal=False)
    assert c.status() == 0
    tol = want * ((pages_a_piece + 64) * 2.0 ** -22 + torch.finfo(q.dtype).eps / 2)
    worst = ((out[:, 0].double() - want).abs() / tol).max().item()
    assert worst <= 1, worst


def test_offsets_beyond_32_bits(kv8, torch):
    """Pages whose byte offsets pass 2^32: written, read, copied and moved there."""
    pages, layers, kvh, dim = 20000, 4, 16, 128      # 256 KB each: 5.2 GB
    c = kv8.Cache.empty(pages, layers, kvh, dim, "int8")
    c.refs[:] = 0
    last = list(range(pages - 6, pages))
    s = kv8.Seqs(dev([last[:3], last[3:]]), dev([40, 40]))
    c.refs[pages - 6:] = 1
    x = torch.randn(80, kvh, dim, device="cuda")
    c.append(3, s, x, x * 2, row_start=dev([0, 40, 80]), max_rows=40)
    assert c.status() == 0
    k, v = c.values(3, s, 1)
    assert float((k - x[40:]).abs().max()) <= 0.04 and float((v - 2 * x[40:]).abs().max()) <= 0.08   # half steps of 2^-4 at most
    for rows in (1, 40):
        q = torch.randn(2 * rows, kvh, dim, device="cuda")
        st = dev([0, rows, 2 * rows])
        a = c.attend(3, s, q, row_start=st, max_rows=rows)
        live = dev([0])
        t2, r2 = torch.full_like(s.table, -1), torch.zeros_like(c.refs)
        c.compact(s, r2, t2, n_live=live)
        assert t2.tolist() == [[0, 1, 2], [3, 4, 5]] and int(live) == 6 and r2[:6].tolist() == [1] * 6
        b = c.attend(3, kv8.Seqs(t2, s.lens), q, row_start=st, max_rows=rows)
        assert torch.equal(a, b)
    c.copy_pages(dev([0]), dev([pages - 7]))
    assert c.status() == 0 and torch.equal(c.codes[pages - 7], c.codes[0])


# ---- pages ---------------------------------------------------------------------------------------------------------
def pool(kv8, pages, seqs, width, seed, layers=2, kvh=2, dim=64, fmt="int8", share=True):
    """A pool in use: sequences of random lengths over random pages, some sharing their first pages."""
    import torch
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = rng.permutation(pages).tolist()
    table, lens, refs = [], [], [0] * pages
    for s in range(seqs):
        n = int(rng.integers(0, (width - 1) * ROWS))
        need = ref.pages_of(n)
        k = int(rng.integers(0, min(need, ref.pages_of(lens[-1])) + 1)) if share and s % 3 == 2 else 0
        k = min(k, n // ROWS, lens[-1] // ROWS if lens else 0)
        if len(order) < need - k:
            n = need = k = 0
        row = (table[-1][:k] if k else []) + [order.pop() for _ in range(need - k)]
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (width - need))
        lens.append(n)
    shape = (pages, layers, 2, kvh)
    c = kv8.Cache(random_codes(shape + (ROWS, dim), fmt, gen), torch.rand(shape, device="cuda", generator=gen),
                  dev(refs), fmt)
    return c, kv8.Seqs(dev(table), dev(lens)), table, lens, refs


@pytest.mark.parametrize("pages,seqs,width", [(60, 1, 5), (300, 40, 9), (9000, 1500, 8)])
def test_reserve(kv8, pages, seqs, width):
    c, s, table, lens, refs = pool(kv8, pages, seqs, width, pages)
    rng = np.random.default_rng(1)
    for step in range(4):
        add = rng.integers(0, [2, 20, 40, 200][step], seqs).tolist()
        if step == 2:
            add[seqs // 2] = -1
        none, bad = ref.reserve(table, lens, refs, add, width)
        c.reserve(s, dev(add))
        got = c.status()
        assert got in ({NO_PAGE, BAD_ARG} if none and bad else {NO_PAGE} if none else {BAD_ARG} if bad else {0})
        assert s.table.tolist() == table and s.lens.tolist() == lens and c.refs.tolist() == refs


@pytest.mark.parametrize("pages,seqs,width,kids", [(40, 1, 4, 1), (500, 30, 9, 64), (9000, 1200, 9, 2100), (120, 12, 9, 60)])
def test_fork(kv8, torch, pages, seqs, width, kids):
    c, s, table, lens, refs = pool(kv8, pages, seqs, width, kids)
    rng = np.random.default_rng(2)
    parents = rng.integers(-1, seqs + (1 if kids == 64 else 0), kids).tolist()    # 64: one parent that is not there
    t2, l2 = [[-7] * (width + 1) for _ in range(kids)], [5] * kids
    d = kv8.Seqs(dev(t2), dev(l2))
    codes, scales = c.codes.clone(), c.scales.clone()
    copies = ref.fork(table, lens, refs, parents, t2, l2)
    c.fork(s, dev(parents), d)
    left_out = any(0 <= q < seqs and lens[q] > 0 and l2[i] == 0 for i, q in enumerate(parents))
    assert c.status() in ({0} if not left_out and max(parents) < seqs else {BAD_ARG, NO_PAGE})
    assert d.lens.tolist() == l2 and c.refs.tolist() == refs
    for i, r in enumerate(d.table.tolist()):
        assert r[:ref.pages_of(l2[i])] == t2[i][:ref.pages_of(l2[i])]
        assert r[ref.pages_of(l2[i]):] == [-7] * (width + 1 - ref.pages_of(l2[i])) or l2[i] == 0
    for a, b in copies:
        codes[b], scales[b] = codes[a], scales[a]
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
    assert s.table.tolist() == table and s.lens.tolist() == lens


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16, 2 ** 30, 5 * ROWS + 1, 4 * ROWS + 1])
def test_fork_leaves_out_lengths_beyond_the_tables(kv8, torch, length):
    """A parent's length that its table, or the child's, does not hold: the child ends empty, the others do not."""
    c = kv8.Cache.empty(40, 1, 1, 64, "int8")
    s, d = kv8.Seqs.empty(2, 5), kv8.Seqs(dev([[-7] * 4] * 2), dev([0, 0]))
    c.reserve(s, dev([20, 20]))
    s.lens[0] = length
    refs = c.refs.tolist()
    c.fork(s, dev([0, 1]), d)
    assert c.status() == BAD_ARG and d.lens.tolist() == [0, 20] and d.table[0].tolist() == [-7] * 4
    full, free = s.table[1, 0].item(), refs.index(0)
    assert d.table[1].tolist() == [full, free, -7, -7]
    refs[full], refs[free] = 2, 1
    assert c.refs.tolist() == refs


def test_free_and_its_indices(kv8):
    c, s, table, lens, refs = pool(kv8, 400, 50, 9, 5)
    which = [3, 7, 3, 49, 0, 7]
    ref.release(table, lens, refs, dict.fromkeys(which))
    c.free(s, dev(which))
    assert c.status() == 0 and s.lens.tolist() == lens and c.refs.tolist() == refs and s.table.tolist() == table
    c.free(s, dev([50, -1, 5]))
    ref.release(table, lens, refs, [5])
    assert c.status() == BAD_ARG and s.lens.tolist() == lens and c.refs.tolist() == refs
    c.free(s)
    assert c.status() == 0 and c.refs.tolist() == [0] * 400 and s.lens.tolist() == [0] * 50
    s.lens[0] = 40
    s.table[0, :3] = dev([1, 1, 400])                       # nobody holds them; one is not there
    c.free(s)
    assert c.status() == BAD_ARG and c.refs.tolist() == [0] * 400
    c.free(s, dev([]).int())


@pytest.mark.parametrize("length", [9 * ROWS + 1, 2 ** 30 + 1, 2 ** 31 - 16, 2 ** 31 - 1])
def test_page_operators_leave_out_lengths_beyond_the_table(kv8, torch, length):
    """Such a sequence stays as it is (status); the others are served."""
    def start():
        c, s, table, lens, refs = pool(kv8, 400, 20, 9, 5, share=False)
        s.lens[7] = length
        s.table[7] = torch.arange(9, dtype=torch.int32, device="cuda")     # whatever lies there is not its own
        table[7] = list(range(9))
        return c, s, table, lens[:7] + [length] + lens[8:], refs

    c, s, table, lens, refs = start()
    ref.release(table, lens, refs, [i for i in range(20) if i != 7])
    c.free(s)
    assert c.status() == BAD_ARG and s.lens.tolist() == lens and c.refs.tolist() == refs
    c.free(s, dev([7, 7]))
    assert c.status() == BAD_ARG and s.lens.tolist() == lens and c.refs.tolist() == refs

    c, s, table, lens, refs = start()
    short = lens[:7] + [0] + lens[8:]
    ref.trim(table, short, refs, 20, 0)
    c.trim(s, 20, 0)
    assert c.status() == BAD_ARG and s.table.tolist() == table and c.refs.tolist() == refs and s.lens.tolist() == lens

    c, s, table, lens, refs = start()
    new_table, new_refs, _, _ = ref.compact(table, lens[:7] + [0] + lens[8:], refs)
    c.compact(s)
    assert c.status() == BAD_ARG and s.table.tolist() == new_table and c.refs.tolist() == new_refs

    c, s, table, lens, refs = start()
    c.reserve(s, dev([0] * 7 + [5] + [0] * 12))
    assert c.status() == BAD_ARG and s.table.tolist() == table and c.refs.tolist() == refs and s.lens.tolist() == lens


def test_empty_lists_do_nothing(kv8, torch):
    """An empty list of sequences or pages is not the C interface's NULL, which means all."""
    c, s, table, lens, refs = pool(kv8, 400, 50, 9, 5)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    c.free(s, none)
    c.copy_pages(none, none)
    assert c.status() == 0 and s.lens.tolist() == lens and c.refs.tolist() == refs


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (16, 16), (33, 17), (10000, 0), (5, 10000)])
def test_trim(kv8, window, sinks):
    c, s, table, lens, refs = pool(kv8, 400, 50, 9, 6)
    for _ in range(2):                                     # the second time there is nothing left to release
        ref.trim(table, lens, refs, window, sinks)
        c.trim(s, window, sinks)
        assert c.status() == 0 and s.table.tolist() == table and c.refs.tolist() == refs and s.lens.tolist() == lens
    ref.release(table, lens, refs, range(50))
    c.free(s)
    assert c.status() == 0 and c.refs.tolist() == refs


@pytest.mark.parametrize("pages,seqs,width", [(7, 1, 4), (200, 20, 9), (9000, 900, 9), (5000, 0, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(kv8, torch, pages, seqs, width, in_place):
    c, s, table, lens, refs = pool(kv8, pages, max(seqs, 1), width, pages + 1)
    if not seqs:
        s.lens.zero_(); c.refs.zero_()
        lens, refs = [0], [0] * pages
    codes, scales = c.codes.clone(), c.scales.clone()
    new_table, new_refs, move, L = ref.compact(table, lens, refs)
    live = dev([-1])
    if in_place:
        c.compact(s, n_live=live)
        t, r = s.table, c.refs
    else:
        t, r = s.table.clone(), torch.full_like(c.refs, 99)
        c.compact(s, r, t, n_live=live)
        assert s.table.tolist() == table and c.refs.tolist() == refs
    assert c.status() == 0 and int(live) == L and t.tolist() == new_table and r.tolist() == new_refs
    for a, b in move.items():
        codes[b], scales[b] = codes[a], scales[a]
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)


def test_compact_full_pool(kv8, torch):
    c = kv8.Cache.empty(64, 1, 1, 64, "int8")
    s = kv8.Seqs(dev([list(range(63, -1, -1))]), dev([1024]))
    c.refs.fill_(1)
    live = dev([0])
    c.compact(s, n_live=live)
    assert c.status() == 0 and int(live) == 64 and s.table[0].tolist() == list(range(63, -1, -1))


def test_copy_pages(kv8, torch):
    c, *_ = pool(kv8, 100, 10, 5, 8)
    codes, scales = c.codes.clone(), c.scales.clone()
    a, b = [3, 3, 50, 99], [4, 5, 0, 98]
    for x, y in zip(a, b):
        codes[y], scales[y] = codes[x], scales[x]
    c.copy_pages(dev(a), dev(b))
    assert c.status() == 0 and torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
    # outside the pool; a destination twice; a destination that is a source: not copied, the others are
    a, b = [1, 2, 7, 8, 100, 10, 11, 12], [20, 20, 21, 7, 22, -1, 11, 23]
    codes[21], scales[21] = codes[7], scales[7]
    codes[23], scales[23] = codes[12], scales[12]
    c.copy_pages(dev(a), dev(b))
    assert c.status() == BAD_ARG and torch.equal(c.codes, codes) and torch.equal(c.scales, scales)


# ---- together ------------------------------------------------------------------------------------------------------
def test_python_checks_arguments(kv8, torch):
    c, s, *_ = make(kv8, "int8", [40, 20], 2, 64)
    q, k = torch.randn(2, 4, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    bad = [lambda: c.attend(2, s, q), lambda: c.attend(0, s, q.double()), lambda: c.attend(0, s, q[:, :3]),
           lambda: c.attend(0, s, q.transpose(0, 1)), lambda: c.attend(0, s, q[:1]), lambda: c.attend(0, s, q, max_rows=2),
           lambda: c.attend(0, s, q, out=q.bfloat16()), lambda: c.attend(0, s, q.cpu()),
           lambda: c.attend(0, s, q, row_start=dev([0, 1])), lambda: c.append(0, s, k, k.bfloat16()),
           lambda: c.append(0, s, k[..., :32], k[..., :32]), lambda: c.reserve(s, dev([1])),
           lambda: c.reserve(s, dev([1, 1]).long()), lambda: c.copy_pages(dev([1]), dev([1, 2])),
           lambda: c.fork(s, dev([0]), s), lambda: kv8.Seqs(s.table, dev([1])), lambda: kv8.Cache(c.codes, c.scales, fmt="x"),
           lambda: kv8.Cache(c.codes[..., :32], c.scales), lambda: kv8.Cache(c.codes, c.scales[:1])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    for f in (lambda: c.attend(0, s, q, causal=False, window=4), lambda: c.attend(0, s, q, scale=0.0),
              lambda: c.trim(s, 0), lambda: c.fork(s, dev([0, 0]), s)):
        with pytest.raises(kv8.KV8Error) as e:
            f()
        assert e.value.code == -1


def test_python_refuses_numbers_beyond_32_bits(kv8, torch):
    """The C interface takes 32-bit integers: 2^32 must not arrive as 0, nor a row stride lose its top."""
    c, s, *_ = make(kv8, "int8", [400, 20], 1, 64)
    q, big = torch.randn(2, 1, 64, device="cuda"), 1 << 32
    refs, table = c.refs.clone(), s.table.clone()
    far = torch.empty_strided((2, 1, 64), (big + 64, 64, 1), dtype=torch.bfloat16, device="cuda")
    st = dev([0, 1, 2])
    bad = [lambda: c.attend(0, s, q, window=big), lambda: c.attend(0, s, q, window=16, sinks=big + 1),
           lambda: c.attend(0, s, q, max_len=big + 400), lambda: c.attend(0, s, q, row_start=st, max_rows=big + 1),
           lambda: c.attend(0, s, q, window=-big), lambda: c.attend(0, s, far), lambda: c.append(0, s, far, far),
           lambda: c.append(0, s, q, q, row_start=st, max_rows=big + 1), lambda: c.attend_workspace(s, q, max_len=big + 400),
           lambda: c.trim(s, big + 1), lambda: c.trim(s, 16, big)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    assert c.status() == 0 and torch.equal(c.refs, refs) and torch.equal(s.table, table)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_values_of_released_pages_are_nan(kv8, torch, fmt):
    """Not those of whatever page a table entry of -1 (or one outside the pool) happens to index."""
    c, s, rc, table = make(kv8, fmt, [70, 20], 2, 64)
    want = c.values(1, s, 0)
    s.table[0, 1], s.table[0, 3] = -1, c.n_pages
    for got, w in zip(c.values(1, s, 0), want):
        gone = torch.zeros(70, dtype=torch.bool, device="cuda")
        gone[16:32] = gone[48:64] = True
        assert got.shape == w.shape and bool(got[gone].isnan().all()) and torch.equal(got[~gone], w[~gone])


def test_python_refuses_a_misaligned_pool(kv8, torch):
    arena = torch.zeros(2 * 2 * ROWS * 64 + 16, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, 1, 2, 1, device="cuda")
    for at in (1, 4, 8):
        with pytest.raises(ValueError):
            kv8.Cache(arena[at:at + 2 * 2 * ROWS * 64].view(2, 1, 2, 1, ROWS, 64), scales)
    kv8.Cache(arena[16:].view(2, 1, 2, 1, ROWS, 64), scales)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_beam_search_run(kv8, torch, fmt):
    """Prompts, then steps of reserve / append / attend / fork / free / trim / compact as a beam search makes them,
    every state and output against the definitions."""
    L, kvh, H, D, pages, width, groups, beams = 2, 2, 4, 64, 400, 12, 3, 3
    n, window, sinks = groups * beams, 60, 3
    c = kv8.Cache.empty(pages, L, kvh, D, fmt)
    a, b = kv8.Seqs.empty(n, width), kv8.Seqs.empty(n, width)
    rc = ref.Cache(to_values(c.codes, fmt), c.scales.cpu().numpy().astype(np.float64), c.refs.cpu().numpy(), fmt)
    table, lens, refs = a.table.tolist(), a.lens.tolist(), c.refs.tolist()
    rng = np.random.default_rng(7)
    gen = torch.Generator(device="cuda").manual_seed(7)
    for step in range(30):
        add = [[37, 0, 50][i // beams] if i % beams == 0 else 0 for i in range(n)] if step == 0 else \
            [int(lens[i] > 0) for i in range(n)]
        if step == 5:                                      # another utterance joins a running batch
            add[beams] = 21
        c.reserve(a, dev(add))
        assert ref.reserve(table, lens, refs, add, width) == (False, False)
        st = starts_of(add)
        for layer in range(L):
            k, v = (torch.randn(max(st[-1], 1), kvh, D, device="cuda", generator=gen) * (1 + step % 4) for _ in (0, 1))
            q = torch.randn(max(st[-1], 1), H, D, device="cuda", generator=gen)
            c.append(layer, a, k, v, row_start=dev(st), max_rows=max(add))
            rc.append(layer, table, lens, k.cpu().numpy(), v.cpu().numpy(), st)
            o = c.attend(layer, a, q, row_start=dev(st), max_rows=max(add), window=window, sinks=sinks)
            want, mass, reach, total = ref.attend(rc, layer, table, lens, q.cpu().numpy(), st, kvh, D ** -0.5, True, window, sinks)
            got = o[:st[-1]].cpu().numpy()
            assert (np.abs(got - want[:st[-1]]) <= tolerance(want, mass, reach, total, D, width, "float32", False)[:st[-1]]).all()
        c.trim(a, window, sinks)
        ref.trim(table, lens, refs, window, sinks)
        parents = [g * beams + int(rng.integers(0, beams)) if step else g * beams for g in range(groups) for _ in range(beams)]
        parents = [q if lens[q] > 0 else -1 for q in parents]
        t2, l2 = b.table.tolist(), [0] * n
        for x, y in ref.fork(table, lens, refs, parents, t2, l2):
            rc.v[y], rc.s[y] = rc.v[x], rc.s[x]
        c.fork(a, dev(parents), b)
        ref.release(table, lens, refs, range(n))
        c.free(a)
        assert b.table.tolist() == t2 and b.lens.tolist() == l2 and c.refs.tolist() == refs
        a, b, table, lens = b, a, t2, l2
        if step % 10 == 9:
            new_table, refs, move, _ = ref.compact(table, lens, refs)
            for x, y in move.items():
                rc.v[y], rc.s[y] = rc.v[x], rc.s[x]
            c.compact(a)
            table = new_table
            assert a.table.tolist() == table and c.refs.tolist() == refs
        assert c.status() == 0
    same_cache(c, rc)
    c.free(a)
    assert c.refs.tolist() == [0] * pages


def test_captured_decode_steps(kv8, torch):
    """A decode step captured once and replayed, two of them with workspaces of their own, on other streams:
    the same bits as the same calls made one by one."""
    kvh, H, D, n, width = 2, 4, 128, 5, 130

    def state(seed):
        c = kv8.Cache.empty(700, 1, kvh, D, "e4m3")
        s = kv8.Seqs.empty(n, width)
        c.reserve(s, dev([2000, 300, 17, 0, 900]))
        x = torch.randn(3217, kvh, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        c.append(0, s, x, x, row_start=dev([0, 2000, 2300, 2317, 2317, 3217]), max_rows=2000)
        add = dev([1, 1, 1, 0, 1])
        k, q = torch.zeros(n, kvh, D, device="cuda"), torch.zeros(n, H, D, device="cuda")
        out = torch.zeros(n, H, D, device="cuda")
        ws, pw = c.attend_workspace(s, q, window=512, sinks=4), c.pages_workspace(s)

        def step():
            c.reserve(s, add, ws=pw)
            c.append(0, s, k, k)
            c.attend(0, s, q, window=512, sinks=4, out=out, ws=ws)
            c.trim(s, 512, 4)
        return c, s, k, q, out, step

    inputs = [(torch.randn(n, kvh, D, device="cuda"), torch.randn(n, H, D, device="cuda")) for _ in range(20)]
    want = []
    c, s, k, q, out, step = state(1)
    for x, y in inputs:
        k.copy_(x); q.copy_(y)
        step()
        want.append(out.clone())
    final = (s.table.tolist(), s.lens.tolist(), c.refs.tolist())
    assert c.status() == 0
    runs = []
    for _ in range(2):
        r = state(1)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            r[5]()
        runs.append((r, stream, g, []))
    torch.cuda.synchronize()
    for x, y in inputs:
        for r, stream, g, got in runs:
            with torch.cuda.stream(stream):
                r[2].copy_(x); r[3].copy_(y)
                g.replay()
                got.append(r[4].clone())
    torch.cuda.synchronize()
    for r, _, _, got in runs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (r[1].table.tolist(), r[1].lens.tolist(), r[0].refs.tolist()) == final
        assert r[0].status() == 0
