"""CPU checks of the 8-bit cache's entry points (include/ct_kv8.h): what they refuse before any CUDA call, the
struct layouts of the ctypes side, and the tests' own 64-bit definitions against hand-worked values."""
import ctypes
import importlib
import os
import subprocess

import numpy as np
import pytest

import kv8_ref as ref

CT_EINVAL, CT_ENOMEM = -1, -2
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def abi():
    return importlib.import_module("cohere-transcribe_b200.abi")


@pytest.fixture(scope="module")
def lib(abi):
    return abi.load()


class Args:
    """Valid arguments that no kernel ever sees: one field at a time is made bad."""

    def __init__(self, abi):
        self.buf = (ctypes.c_uint8 * 8192)()
        self.a = (ctypes.addressof(self.buf) + 255) // 256 * 256
        self.abi = abi

    def cache(self, **kw):
        d = dict(codes=self.a, scales=self.a, refs=self.a, n_pages=4, n_layers=2, kv_heads=2, head_dim=64, format=0)
        d.update(kw)
        return self.abi.KV8Cache(*[d[f] for f, _ in self.abi.KV8Cache._fields_])

    def seqs(self, table=None, **kw):
        d = dict(table=self.a if table is None else table, len=self.a, n_seqs=3, table_stride=4)
        d.update(kw)
        return self.abi.KV8Seqs(*[d[f] for f, _ in self.abi.KV8Seqs._fields_])


@pytest.fixture
def args(abi):
    return Args(abi)


BAD_CACHES = [dict(codes=None), dict(scales=None), dict(n_pages=0), dict(n_layers=0), dict(kv_heads=0),
              dict(kv_heads=5000), dict(head_dim=96), dict(head_dim=0), dict(format=2), dict(format=-1)]
BAD_SEQS = [dict(len=None), dict(n_seqs=0), dict(n_seqs=65536), dict(table_stride=0)]


def _append(lib, args, cache=None, seqs=None, **kw):
    d = dict(layer=0, k=args.a, ldk=128, v=args.a, ldv=128, type=0, n_rows=9, rs=args.a, max_rows=4)
    d.update(kw)
    c = args.cache() if cache is None else cache
    s = args.seqs() if seqs is None else seqs
    return lib.ct_kv8_append(ctypes.byref(c), d["layer"], ctypes.byref(s), d["k"], d["ldk"], d["v"], d["ldv"], d["type"],
                             d["n_rows"], d["rs"], d["max_rows"], None)


def _attn(lib, args, cache=None, seqs=None, **kw):
    d = dict(layer=0, q=args.a, ldq=256, out=args.a, ldo=256, type=0, n_rows=9, rs=args.a, max_rows=4, max_len=64,
             heads=4, scale=0.1, causal=1, window=0, sinks=0, ws=None, ws_bytes=0)
    d.update(kw)
    c = args.cache() if cache is None else cache
    s = args.seqs() if seqs is None else seqs
    return lib.ct_kv8_attn(ctypes.byref(c), d["layer"], ctypes.byref(s), d["q"], d["ldq"], d["out"], d["ldo"], d["type"],
                           d["n_rows"], d["rs"], d["max_rows"], d["max_len"], d["heads"], d["scale"], d["causal"],
                           d["window"], d["sinks"], d["ws"], d["ws_bytes"], None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(lib, args, bad):
    c, s = args.cache(**bad), args.seqs()
    assert _append(lib, args, cache=c) == CT_EINVAL
    assert _attn(lib, args, cache=c) == CT_EINVAL
    r, p = ctypes.byref(c), ctypes.byref(s)
    t = ctypes.byref(args.seqs(table=args.a + 256, len=args.a + 512))
    assert lib.ct_kv8_reserve(r, p, args.a, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_fork(r, p, args.a, t, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_free(r, p, None, 0, None) == CT_EINVAL
    assert lib.ct_kv8_trim(r, p, 16, 0, None) == CT_EINVAL
    assert lib.ct_kv8_compact(r, p, args.a, args.a, None, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_copy_pages(r, args.a, args.a, 1, None) == CT_EINVAL
    assert lib.ct_kv8_pages_ws_bytes(r, 3) == 0


@pytest.mark.parametrize("bad", BAD_SEQS + [dict(table=0)], ids=str)
def test_bad_sequences_are_refused(lib, args, bad):
    c, s = args.cache(), args.seqs(**bad)
    if bad.get("table") == 0:
        s.table = None
    assert _append(lib, args, seqs=s) == CT_EINVAL
    assert _attn(lib, args, seqs=s) == CT_EINVAL
    r, p = ctypes.byref(c), ctypes.byref(s)
    assert lib.ct_kv8_reserve(r, p, args.a, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_free(r, p, None, 0, None) == CT_EINVAL
    assert lib.ct_kv8_trim(r, p, 16, 0, None) == CT_EINVAL
    assert lib.ct_kv8_compact(r, p, args.a, args.a, None, args.a, 4096, None) == CT_EINVAL


@pytest.mark.parametrize("field,offset", [("codes", 1), ("codes", 8), ("scales", 1), ("scales", 2)])
def test_misaligned_pools_are_refused(lib, args, field, offset):
    """codes by 16 bytes, scales by 4: the kernels read them that wide."""
    c, s = args.cache(**{field: args.a + offset}), args.seqs()
    assert _append(lib, args, cache=c) == CT_EINVAL
    assert _attn(lib, args, cache=c) == CT_EINVAL
    r, p = ctypes.byref(c), ctypes.byref(s)
    t = ctypes.byref(args.seqs(table=args.a + 256, len=args.a + 512))
    assert lib.ct_kv8_pages_ws_bytes(r, 3) == 0
    assert lib.ct_kv8_attn_ws_bytes(r, p, 0, 9, 4, 64, 4, 1, 0, 0) == 0
    assert lib.ct_kv8_reserve(r, p, args.a, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_fork(r, p, args.a, t, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_free(r, p, None, 0, None) == CT_EINVAL
    assert lib.ct_kv8_trim(r, p, 16, 0, None) == CT_EINVAL
    assert lib.ct_kv8_compact(r, p, args.a, args.a, None, args.a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_copy_pages(r, args.a, args.a, 1, None) == CT_EINVAL


@pytest.mark.parametrize("bad", [
    dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(ldk=127), dict(ldv=126), dict(ldk=130),
    dict(type=2), dict(n_rows=0), dict(max_rows=0), dict(max_rows=(1 << 20) + 1), dict(rs=None),
    dict(rs=None, max_rows=1, n_rows=2)], ids=str)
def test_append_refuses(lib, args, bad):
    assert _append(lib, args, **bad) == CT_EINVAL
    assert _append(lib, args, k=args.a + 8) == CT_EINVAL


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(q=None), dict(out=None), dict(ldq=252), dict(ldo=255), dict(type=3), dict(n_rows=0),
    dict(max_rows=0), dict(max_len=0), dict(max_len=(1 << 30) + 1), dict(heads=3), dict(heads=0), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-1),
    dict(causal=0, window=8), dict(rs=None), dict(rs=None, max_rows=1, n_rows=2)], ids=str)
def test_attention_refuses(lib, args, bad):
    assert _attn(lib, args, **bad) == CT_EINVAL


def test_attention_checks_its_workspace(lib, args):
    c, s = args.cache(n_pages=1000), args.seqs(n_seqs=1, table_stride=1000)
    r, p = ctypes.byref(c), ctypes.byref(s)
    need = lib.ct_kv8_attn_ws_bytes(r, p, 0, 1, 1, 16000, 4, 1, 0, 0)
    assert need > 0
    kw = dict(cache=c, seqs=s, n_rows=1, rs=None, max_rows=1, max_len=16000)
    assert _attn(lib, args, ws=None, ws_bytes=need, **kw) == CT_EINVAL
    assert _attn(lib, args, ws=args.a, ws_bytes=need - 1, **kw) == CT_ENOMEM
    assert lib.ct_kv8_attn_ws_bytes(r, p, 7, 1, 1, 16000, 4, 1, 0, 0) == 0


def test_page_operators_refuse(lib, args):
    c, s = args.cache(), args.seqs()
    r, p, a = ctypes.byref(c), ctypes.byref(s), args.a
    no_refs = ctypes.byref(args.cache(refs=None))
    t = ctypes.byref(args.seqs(table=a + 256, len=a + 512))
    assert lib.ct_kv8_reserve(no_refs, p, a, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_fork(no_refs, p, a, t, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_free(no_refs, p, None, 0, None) == CT_EINVAL
    assert lib.ct_kv8_trim(no_refs, p, 16, 0, None) == CT_EINVAL
    assert lib.ct_kv8_compact(no_refs, p, a, a, None, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_reserve(r, p, None, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_reserve(r, p, a, None, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_reserve(r, p, a, a + 4, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_reserve(r, p, a, a, 8, None) == CT_ENOMEM
    assert lib.ct_kv8_fork(r, p, a, p, a, 4096, None) == CT_EINVAL          # dst is src
    assert lib.ct_kv8_fork(r, p, None, t, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_fork(r, p, a, t, a, 8, None) == CT_ENOMEM
    assert lib.ct_kv8_free(r, p, a, -1, None) == CT_EINVAL
    assert lib.ct_kv8_trim(r, p, 0, 0, None) == CT_EINVAL
    assert lib.ct_kv8_trim(r, p, 16, -1, None) == CT_EINVAL
    assert lib.ct_kv8_compact(r, p, None, a, None, a, 4096, None) == CT_EINVAL
    assert lib.ct_kv8_compact(r, p, a, a, None, a, 8, None) == CT_ENOMEM
    assert lib.ct_kv8_copy_pages(r, None, a, 1, None) == CT_EINVAL
    assert lib.ct_kv8_copy_pages(r, a, a, 4097, None) == CT_EINVAL
    assert lib.ct_kv8_copy_pages(r, a, a, -1, None) == CT_EINVAL
    assert lib.ct_kv8_pages_ws_bytes(r, 0) == 0 and lib.ct_kv8_pages_ws_bytes(r, 65536) == 0


@pytest.mark.parametrize("table,length", [(0, 512), (16, 512), (32, 512), (44, 512), (-44, 512), (256, 0), (256, 8), (256, -8)])
def test_fork_refuses_sequences_that_overlap(lib, args, table, length):
    """dst's table or lengths inside src's: three rows of four entries, three lengths."""
    c, a = args.cache(), args.a + 1024
    s, d = args.seqs(table=a, len=a + 2048), args.seqs(table=a + table, len=a + 2048 + length)
    assert lib.ct_kv8_fork(ctypes.byref(c), ctypes.byref(s), args.a, ctypes.byref(d), args.a, 4096, None) == CT_EINVAL
    for t, n in ((48, 12), (-48, -12)):                        # side by side: taken
        d = args.seqs(table=a + t, len=a + 2048 + n)
        assert lib.ct_kv8_fork(ctypes.byref(c), ctypes.byref(s), args.a, ctypes.byref(d), args.a, 8, None) == CT_ENOMEM


def test_reserve_refuses_tables_whose_pages_do_not_count_in_32_bits(lib, args):
    """The pages that all sequences ask for are summed in 32 bits."""
    c, a = args.cache(), args.a
    for n, stride in ((32, 1 << 26), (65535, 1 << 16), (65535, 1 << 26)):
        s = args.seqs(n_seqs=n, table_stride=stride)
        assert lib.ct_kv8_reserve(ctypes.byref(c), ctypes.byref(s), a, a, 1 << 20, None) == CT_EINVAL
    s = args.seqs(n_seqs=31, table_stride=1 << 26)
    assert lib.ct_kv8_reserve(ctypes.byref(c), ctypes.byref(s), a, a, 8, None) == CT_ENOMEM     # taken


def test_ctypes_structs_match_the_header(abi, tmp_path):
    src = tmp_path / "o.c"
    fields = [("ct_kv8_cache", f) for f, _ in abi.KV8Cache._fields_] + [("ct_kv8_seqs", f) for f, _ in abi.KV8Seqs._fields_]
    src.write_text('#include <stdio.h>\n#include "ct_kv8.h"\nint main(void) {\n' + "".join(
        f'printf("%zu ", offsetof({t}, {f}));\n' for t, f in fields) +
        'printf("%zu %zu %d\\n", sizeof(ct_kv8_cache), sizeof(ct_kv8_seqs), CT_KV8_ROWS); return 0; }\n')
    exe = tmp_path / "o"
    subprocess.run(["gcc", f"-I{os.path.join(REPO, 'include')}", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    types = {"ct_kv8_cache": abi.KV8Cache, "ct_kv8_seqs": abi.KV8Seqs}
    assert got == [getattr(types[t], f).offset for t, f in fields] + [ctypes.sizeof(abi.KV8Cache),
                                                                     ctypes.sizeof(abi.KV8Seqs), ref.ROWS]


def test_reference_rounding():
    """Hand-worked codes: E4M3 has 3 mantissa bits, steps of 2^-9 below 2^-6, ties to even, largest 448."""
    assert ref.nearest([1.0, 1.0625, 1.1875, 449.0, 2.0 ** -10, 3 * 2.0 ** -10, -0.3], "e4m3").tolist() == \
        [1.0, 1.0, 1.25, 448.0, 0.0, 2.0 ** -8, -0.3125]
    assert ref.nearest([0.5, 1.5, -2.5, 127.4, 300.0], "int8").tolist() == [0.0, 2.0, -2.0, 127.0, 127.0]
    assert ref.block_scale(448.0, "e4m3") == 1.0 and ref.block_scale(448.1, "e4m3") == 2.0
    assert ref.block_scale(127.0, "int8") == 1.0 and ref.block_scale(63.5, "int8") == 0.5
    assert ref.block_scale(0.0, "int8") == 2.0 ** -126


def test_reference_attention_of_one_key_is_its_value():
    rng = np.random.default_rng(0)
    c = ref.Cache(rng.integers(-127, 128, (2, 1, 2, 1, 16, 64)).astype(float), np.full((2, 1, 2, 1), 0.25),
                  np.ones(2, int), "int8")
    q = rng.standard_normal((2, 1, 64))
    out, mass, _, _ = ref.attend(c, 0, [[1, 0]], [2], q, [0, 2], 1, 0.125)
    assert np.allclose(out[0, 0], c.v[1, 0, 1, 0, 0] * 0.25) and np.allclose(mass[0], np.abs(out[0]))
    out, _, _, _ = ref.attend(c, 0, [[1, 0]], [18], q, [0, 2], 1, 0.125, window=1, sinks=0)
    assert np.allclose(out[:, 0], c.v[0, 0, 1, 0, :2] * 0.25)
