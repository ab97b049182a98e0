"""Checks of a decoder's step over a paged cache without a GPU: the entry points (sfe_decode.cpp) built with
tests/model_ops_stubs.cpp and tests/decode_stubs.cpp in place of a context and its kernels.  Addresses are made up:
nothing reads them."""
import ctypes
import os
import subprocess

import pytest

from scriptrs_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "scriptrs_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
AT = 1 << 24  # an address


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    lib = str(tmp_path_factory.mktemp("checks") / "checks.so")
    subprocess.run([HIPCC, "-O1", "-g", "-std=c++17", "-x", "hip", "--cuda-host-only", "-fPIC", "-shared",
                    "-Wno-unused-command-line-argument", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                    os.path.join(CSRC, "sfe_decode.cpp"), os.path.join(ROOT, "tests", "model_ops_stubs.cpp"),
                    os.path.join(ROOT, "tests", "decode_stubs.cpp"), "-o", lib], check=True, stderr=subprocess.DEVNULL)
    L, real = ctypes.CDLL(lib), _lib.lib()
    for name in _lib.EXPORTS:
        if hasattr(L, name):
            f = getattr(real, name)
            getattr(L, name).argtypes, getattr(L, name).restype = f.argtypes, f.restype
    L.stub_message.restype = ctypes.c_char_p
    L.stub_context.restype = ctypes.c_void_p
    L.stub_destroy.argtypes = [ctypes.c_void_p]
    L.stub_page_of.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                               ctypes.c_int64]
    L.stub_page_of.restype = ctypes.c_int64
    L.stub_attn_whole.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]
    L.stub_attn_tiles.argtypes = [ctypes.c_int64]
    return L


@pytest.fixture
def ctx(checks):
    c = checks.stub_context()
    yield c
    checks.stub_destroy(c)


def passes(L, rc):
    assert rc == _lib.SFE_OK, L.stub_message()


def refused(L, rc, part):
    assert rc == _lib.SFE_INVALID_ARG and part in L.stub_message().decode(), (rc, L.stub_message())


def offsets(*o):
    return (ctypes.c_int64 * len(o))(*o)


def make(L, ctx, new=(0, 1, 3), heads=4, kv_heads=2, dim=64):
    plan = ctypes.c_void_p()
    rc = L.sfe_cache_plan_make(ctx, offsets(*new), len(new) - 1, heads, kv_heads, dim, None, ctypes.byref(plan))
    return rc, plan


def cache(data=AT, pages=4, page=16, kv_heads=2, dim=64, kind=4):
    return _lib.SfeCache(data, pages, page, kv_heads, dim, kind)


def tokens(table=AT - 8192, stride=2, pages=2, lengths=AT - 4096):
    return _lib.SfeCacheTokens(table, stride, pages, lengths)


def heads(data, row=128, head=64):
    return ctypes.byref(_lib.SfeHeads(data, row, head))


def test_records(checks):
    L = checks
    assert L.sfe_cache_record(16, 64, 1) == L.sfe_cache_record(16, 64, 2) == 2 * 16 * 64 * 2
    assert L.sfe_cache_record(64, 128, 3) == L.sfe_cache_record(64, 128, 4) == 2 * 64 * 128 + 8 * 64
    for page, dim, kind, part in ((8, 64, 1, "page_size"), (2048, 64, 1, "page_size"), (48, 64, 1, "page_size"), (16, 8, 1, "head_dim"),
                                  (16, 0, 1, "head_dim"), (16, 144, 1, "head_dim"), (16, 64, 0, "type"), (16, 64, 5, "type")):
        assert L.sfe_cache_record(page, dim, kind) == 0 and part in L.stub_message().decode()


def test_plans(checks, ctx):
    L = checks
    for new, args, part in (((1, 2), {}, "begin at 0"), ((0, 2, 1), {}, "non-decreasing"), ((0, 1), {"heads": 3}, "multiple of kv_heads"),
                            ((0, 1), {"heads": 2048}, "1024"), ((0, 1), {"dim": 40}, "head_dim"), ((0, (1 << 24) + 1), {}, "2^24"),
                            ((0, 1 << 24), {"heads": 64, "kv_heads": 1}, "2^28"), ((-1, 1), {}, "negative")):
        rc, plan = make(L, ctx, new, **args)
        refused(L, rc, part)
        assert not plan.value
    refused(L, make(L, None)[0], "null context")
    rc, plan = make(L, ctx, (0, 0, 0))  # (no new tokens)
    passes(L, rc)
    passes(L, L.sfe_cache_write(plan, ctypes.byref(cache()), ctypes.byref(tokens(0, 0, 0, 0)), 1, heads(0), heads(0), None))
    L.sfe_cache_plan_free(plan)


def test_a_plan_that_outlives_its_context_is_refused(checks):
    L = checks
    ctx = L.stub_context()
    rc, plan = make(L, ctx)
    passes(L, rc)
    L.stub_destroy(ctx)
    refused(L, L.sfe_cache_write(plan, ctypes.byref(cache()), ctypes.byref(tokens()), 1, heads(AT * 2), heads(AT * 2 + 1024), None), "destroyed")
    L.sfe_cache_plan_free(plan)


def test_moves(checks, ctx):
    """3 new tokens, 2 kv heads of 64: rows of 256 bytes in 16 bits; the cache is 4 pages of 2 records of 2,176 bytes."""
    L = checks
    plan = make(L, ctx)[1]
    size = 4 * 2 * (2 * 16 * 64 + 8 * 16)

    def write(c=None, t=None, k=heads(2 * AT), v=heads(2 * AT + 4096), dtype=1):
        return L.sfe_cache_write(plan, ctypes.byref(c or cache()), ctypes.byref(t or tokens()), dtype, k, v, None)

    def read(c=None, t=None, k=heads(2 * AT), v=heads(2 * AT + 4096), dtype=1):
        return L.sfe_cache_read(plan, ctypes.byref(c or cache()), ctypes.byref(t or tokens()), dtype, k, v, None)
    for f in (write, read):
        passes(L, f())
        passes(L, f(dtype=0))
        refused(L, f(dtype=3), "dtype")
        refused(L, f(c=cache(kv_heads=1)), "the plan's")
        refused(L, f(c=cache(dim=128)), "the plan's")
        refused(L, f(c=cache(page=24)), "page_size")
        refused(L, f(c=cache(kind=9)), "type")
        refused(L, f(c=cache(data=0)), "null cache")
        refused(L, f(c=cache(data=AT + 8)), "aligned")
        refused(L, f(c=cache(pages=-1)), "pages")
        refused(L, f(c=cache(pages=1 << 31)), "pages")
        passes(L, f(c=cache(data=0, pages=0)))
        refused(L, f(t=tokens(lengths=0)), "null page_table or lengths")
        refused(L, f(t=tokens(table=0)), "null page_table or lengths")
        passes(L, f(t=tokens(table=0, pages=0)))
        refused(L, f(t=tokens(table=AT - 8190)), "aligned")
        refused(L, f(t=tokens(stride=-1)), "table_stride")
        refused(L, f(t=tokens(pages=-1)), "table_pages")
        refused(L, f(k=heads(0)), "null k")
        refused(L, f(v=heads(2 * AT + 8)), "aligned")
        refused(L, f(k=heads(2 * AT, 132)), "aligned")
        refused(L, f(k=heads(AT + size - 16)), "k overlaps the cache")
        refused(L, f(v=heads(AT - 3 * 256 + 16)), "v overlaps the cache")
        passes(L, f(k=heads(AT + size)))
    passes(L, write(v=heads(2 * AT)))          # (read twice)
    refused(L, read(v=heads(2 * AT)), "k overlaps v")
    passes(L, read(k=heads(2 * AT, 256), v=heads(2 * AT + 256, 256)))  # (halves of one tensor)
    passes(L, write(k=heads(2 * AT, 0, 0)))    # (one row for all)
    refused(L, read(k=heads(2 * AT, 0, 64)), "overlap")
    refused(L, read(k=heads(2 * AT, 64, 64)), "overlap")
    refused(L, read(k=heads(AT - 8192)), "k overlaps page_table")
    refused(L, read(v=heads(AT - 4096)), "v overlaps lengths")
    refused(L, write(t=tokens(table=AT + 16)), "cache overlaps page_table")
    refused(L, write(t=tokens(lengths=AT + size - 4)), "cache overlaps lengths")
    L.sfe_cache_plan_free(plan)


def test_attention(checks, ctx):
    L = checks
    plan = make(L, ctx)[1]

    def attend(c=None, t=None, dtype=1, q=heads(2 * AT, 256), tree=None, scale=0.125, out=heads(3 * AT, 256), rows=3, p=plan):
        return L.sfe_cache_attention(p, ctypes.byref(c or cache()), ctypes.byref(t or tokens()), dtype, q, tree, scale, out, rows, None)
    passes(L, attend())
    passes(L, attend(dtype=2))
    passes(L, attend(rows=10))
    passes(L, attend(tree=4 * AT))
    passes(L, attend(c=cache(kind=1)))
    refused(L, attend(c=cache(kind=1), dtype=2), "the queries' dtype")
    refused(L, attend(dtype=0), "dtype")
    refused(L, attend(rows=2), "rows")
    refused(L, attend(tree=4 * AT + 4), "aligned")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(L, attend(scale=scale), "scale")
    refused(L, attend(q=heads(2 * AT + 2, 256)), "aligned")
    refused(L, attend(out=heads(0, 256)), "null out")
    refused(L, attend(out=heads(2 * AT + 256, 256)), "out overlaps q")
    refused(L, attend(out=heads(AT, 256)), "out overlaps the cache")
    refused(L, attend(out=heads(AT - 8192, 256)), "out overlaps page_table")
    refused(L, attend(tree=3 * AT + 8), "out overlaps tree")
    refused(L, attend(out=heads(3 * AT, 0)), "overlap")
    refused(L, attend(t=tokens(pages=1 << 27)), "2^30")
    passes(L, attend(t=tokens(table=1 << 40, pages=1 << 26)))  # (256 MB a row: far from the others)
    tall = make(L, ctx, (0, 65))[1]
    passes(L, attend(p=tall, rows=65))
    refused(L, attend(p=tall, rows=65, tree=4 * AT), "64 new tokens")
    many = make(L, ctx, tuple(range(2049)))[1]
    refused(L, attend(p=many, rows=2048, t=tokens(pages=1 << 22)), "too large")
    for p in (plan, tall, many):
        L.sfe_cache_plan_free(p)


def test_norm_rotary(checks):
    L, table = checks, _lib.SfeRotaryTable()
    assert _lib.lib().sfe_rotary_init(ctypes.byref(table), 64, 0, 1e4, 0, 1.0, 1.0, 1.0, 32.0, 1.0) == 0
    ctx = ctypes.c_void_p(1)

    def call(norm=2, eps=1e-5, dtype=1, pos=AT, rows=5, dim=64, qh=2, qw=AT * 4, q=heads(AT * 2), qo=heads(AT * 3), kh=1, kw=None,
             k=heads(AT * 5, 64), ko=heads(AT * 6, 64), t=table):
        return L.sfe_norm_rotary(ctx, ctypes.byref(t), norm, eps, dtype, pos, rows, dim, qh, qw, q, qo, kh, kw, k, ko, None)
    passes(L, call())
    passes(L, call(norm=1))
    passes(L, call(qo=heads(AT * 2), ko=heads(AT * 5, 64)))
    passes(L, call(rows=0, pos=None))
    passes(L, call(kh=0, k=None, ko=None))
    refused(L, call(norm=0), "norm must")
    refused(L, call(norm=3), "norm must")
    refused(L, call(eps=-1.0), "eps")
    refused(L, call(eps=float("nan")), "eps")
    refused(L, call(dtype=4), "dtype")
    refused(L, call(rows=-1), "rows")
    refused(L, call(dim=62), "head_dim")
    refused(L, call(dim=258), "head_dim")
    refused(L, call(t=_lib.SfeRotaryTable()), "not initialised")
    refused(L, call(pos=None), "null positions")
    refused(L, call(pos=AT + 2), "positions must be aligned")
    refused(L, call(qw=AT * 4 + 1), "q_weight")
    refused(L, call(q=None), "null q")
    refused(L, call(qo=heads(AT * 2 + 64)), "q_out overlaps q")
    refused(L, call(ko=heads(AT * 2, 64)), "k_out overlaps q")
    refused(L, call(ko=heads(AT * 3 + 128, 64)), "q_out overlaps k_out")
    refused(L, call(qo=heads(AT * 4)), "q_out overlaps q_weight")
    refused(L, call(kw=AT * 3 + 128), "q_out overlaps k_weight")
    refused(L, call(qo=heads(AT - 64)), "q_out overlaps positions")
    refused(L, call(qo=heads(AT * 3, 0)), "overlap")


def test_logits(checks):
    L, ctx = checks, ctypes.c_void_p(1)

    def call(**changes):
        a = _lib.SfeLogits(dtype=1, rows=4, vocab=100, history_most=8, logits=AT, out=AT * 2, logits_row=100, out_row=100, history=AT * 3,
                           history_row=8, lengths=AT * 4, repetition=1.5, presence=0.0, frequency=0.0, bias=AT * 5, bias_row=0,
                           allowed=AT * 6, allowed_row=4, n_allowed=3, states=AT * 7)
        for name, value in changes.items():
            setattr(a, name, value)
        return L.sfe_adjust_logits(ctx, ctypes.byref(a), None)
    passes(L, call())
    passes(L, call(out=AT))
    passes(L, call(rows=0, logits=None))
    passes(L, call(history=None, lengths=None))
    passes(L, call(repetition=0.0, repetitions=AT * 8))
    refused(L, call(dtype=5), "dtype")
    refused(L, call(rows=-1), "rows")
    refused(L, call(vocab=0), "vocab")
    refused(L, call(vocab=(1 << 24) + 1), "vocab")
    refused(L, call(history=None), "lengths without")
    refused(L, call(allowed=None), "states without")
    refused(L, call(history_most=-1), "history_most")
    refused(L, call(history_most=(1 << 30) + 1), "history_most")
    refused(L, call(n_allowed=-1), "n_allowed")
    for value in (0.0, -1.0, float("inf"), float("nan")):
        refused(L, call(repetition=value), "repetition")
    refused(L, call(presence=float("nan")), "presence")
    refused(L, call(frequency=float("inf")), "frequency")
    refused(L, call(logits_row=-1), "strides")
    refused(L, call(bias_row=1 << 41), "strides")
    refused(L, call(out=None), "null")
    refused(L, call(out=AT * 2 + 1), "aligned")
    refused(L, call(history=AT * 3 + 2), "history must be aligned")
    refused(L, call(states=AT * 7 + 1), "states must be aligned")
    refused(L, call(out_row=99), "rows overlap")
    refused(L, call(out=AT + 2), "out overlaps logits")
    refused(L, call(out=AT, out_row=101), "out overlaps logits")
    for name, at in (("history", 3), ("lengths", 4), ("bias", 5), ("allowed", 6), ("states", 7)):
        refused(L, call(out=AT * at), f"out overlaps {name}")
    refused(L, call(frequencies=AT * 2 + 796), "out overlaps frequency")


def test_places(checks):
    """Tokens in no place, without a read past the table: it lies between numbers that would be taken for pages."""
    guarded = (ctypes.c_int32 * 10)(3, 3, 5, 0, 2, -1, 7, 2_147_483_647, 3, 3)
    table = ctypes.addressof(guarded) + 8  # [2][3]

    def page(seq, token):
        return checks.stub_page_of(table, 3, 3, 7, 4, seq, token)
    assert [page(0, t) for t in (0, 15, 16, 31, 32, 47)] == [5, 5, 0, 0, 2, 2]
    assert [page(1, t) for t in (0, 16, 32)] == [-1, -1, -1]
    for token in (-1, -16, -(1 << 40), 48, 63, 1 << 31, (1 << 40) + 1):
        assert page(0, token) == page(1, token) == -1
    assert checks.stub_page_of(None, 0, 0, 7, 4, 0, 0) == -1


def test_tiles_and_shares(checks):
    L = checks
    assert [L.stub_attn_tiles(n) for n in (1, 16, 17, 32, 33, 64, 65, 1 << 24)] == [1, 1, 2, 2, 4, 4, 8, 8]
    assert [L.stub_attn_round(n) for n in (1, 2, 4, 8)] == [128, 128, 64, 32]
    assert L.stub_attn_whole(4, 128, 1, 1) and L.stub_attn_whole(1024, 1875, 1, 1) and L.stub_attn_whole(4, 600, 1, 1)
    assert not L.stub_attn_whole(4, 1200, 1, 1) and not L.stub_attn_whole(4096, 5000, 1, 1) and L.stub_attn_whole(8192, 5000, 1, 1)
    assert not L.stub_attn_whole(8192, 60000, 1, 1) and L.stub_attn_whole(8192, 40000, 8, 1)
