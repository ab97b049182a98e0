"""The model operators' checks of their tensors without a GPU: the entry points (sfe_ops.cpp) built with
tests/model_ops_stubs.cpp in place of a context and its kernels.  Addresses are made up: nothing reads them."""
import ctypes
import os
import subprocess

import pytest

from scriptrs_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "scriptrs_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CTX = ctypes.c_void_p(1)
AT = 1 << 20  # an address


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    lib = str(tmp_path_factory.mktemp("checks") / "checks.so")
    subprocess.run([HIPCC, "-O1", "-g", "-std=c++17", "-x", "hip", "--cuda-host-only", "-fPIC", "-shared",
                    "-Wno-unused-command-line-argument", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                    os.path.join(CSRC, "sfe_ops.cpp"), os.path.join(CSRC, "sfe_attn_plan.cpp"),
                    os.path.join(ROOT, "tests", "model_ops_stubs.cpp"), "-o", lib], check=True, stderr=subprocess.DEVNULL)
    L, real = ctypes.CDLL(lib), _lib.lib()
    for name in _lib.EXPORTS:
        if hasattr(L, name):
            f = getattr(real, name)
            getattr(L, name).argtypes, getattr(L, name).restype = f.argtypes, f.restype
    L.stub_message.restype = ctypes.c_char_p
    return L


def passes(L, rc):
    assert rc == _lib.SFE_OK, L.stub_message()


def refused(L, rc, part):
    assert rc == _lib.SFE_INVALID_ARG and part in L.stub_message().decode(), (rc, L.stub_message())


def reorder(L, *states, streams=2, beams=3, parents=AT - 4096):
    """States (in, out, outer, inner bytes) of streams * beams rows."""
    s = (_lib.SfeBeamState * len(states))(*[_lib.SfeBeamState(*x) for x in states])
    return L.sfe_beam_reorder(CTX, parents, streams, beams, s, len(states), None)


def test_reordered_states_share_no_memory(checks):
    """One launch moves all states: none may write what another reads or writes."""
    L, a, b, c = checks, AT, AT + 600, AT + 1200  # 600 bytes: 6 rows of 100
    passes(L, reorder(L, (a, a, 1, 100), (b, b, 1, 100)))
    passes(L, reorder(L, (a, b, 1, 100)))
    passes(L, reorder(L, (a, b, 1, 100), (a, c, 1, 100)))  # (read twice)
    passes(L, reorder(L, (a, a, 1, 100), (a, a, 0, 100)))  # (the second is empty)
    refused(L, reorder(L, (a, b, 1, 100), (b, a, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, a, 1, 100), (a, a, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, a, 1, 100), (a, b, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, c, 1, 100), (b, c, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, c, 1, 100), (b, c + 599, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, b, 1, 100), (b + 100, c, 1, 100)), "overlaps")
    refused(L, reorder(L, (a, a + 300, 1, 100)), "overlaps")
    refused(L, reorder(L, (b, b, 1, 100), (a, a, 2, 100)), "overlaps")
    many = [(AT + 2000 * i, AT + 2000 * i + 600 * (i % 2), 1, 100) for i in range(50)]
    passes(L, reorder(L, *many))
    refused(L, reorder(L, *many, (AT + 500_000, AT + 2000 * 31 + 900, 1, 100)), "overlaps")


def test_reordered_states_leave_the_parents(checks):
    passes(checks, reorder(checks, (AT, AT, 1, 100), parents=AT + 600))
    refused(checks, reorder(checks, (AT, AT, 1, 100), parents=AT + 596), "overlaps")


def offsets(*o):
    return (ctypes.c_int64 * len(o))(*o)


def make_plan(L, ctx, q=(0, 40, 300), k=(0, 40, 300)):
    plan = ctypes.c_void_p()
    passes(L, L.sfe_attention_plan(ctx, offsets(*q), offsets(*k), len(q) - 1, 2, 2, 64, -1, -1, None, ctypes.byref(plan)))
    return plan


def attend(L, plan):
    x, out = _lib.SfeHeads(AT, 128, 64), _lib.SfeHeads(1 << 30, 128, 64)
    return L.sfe_attention(plan, _lib.SFE_BF16, x, x, x, None, 0.125, out, None)


@pytest.fixture
def contexts(checks):
    checks.stub_context.restype = ctypes.c_void_p
    checks.stub_destroy.argtypes = [ctypes.c_void_p]
    return checks


@pytest.mark.parametrize("q", [(0, 40, 300), (0, 0, 0)], ids=["rows", "none"])
def test_plans_that_outlive_their_context(contexts, q):
    """Refused, and freeing them touches neither the context that is gone nor one made since."""
    L = contexts
    ctx = L.stub_context()
    plan = make_plan(L, ctx, q=q)
    passes(L, attend(L, plan))
    assert L.stub_destroy(ctx) == (1 if q[-1] else 0)
    refused(L, attend(L, plan), "destroyed")
    other = L.stub_context()
    refused(L, attend(L, plan), "destroyed")
    L.sfe_attention_plan_free(plan)
    assert L.stub_destroy(other) == 0


def test_buffers_of_freed_plans_are_reused(contexts):
    L = contexts
    ctx = L.stub_context()
    a, b = make_plan(L, ctx), make_plan(L, ctx)
    L.sfe_attention_plan_free(a)
    c = make_plan(L, ctx)  # (takes a's buffer)
    L.sfe_attention_plan_free(b)
    L.sfe_attention_plan_free(c)
    d = make_plan(L, ctx)
    assert L.stub_destroy(ctx) == 2
    L.sfe_attention_plan_free(d)


def test_rows_of_no_sequence_overlap_nothing(contexts):
    """sfe_attention_rows writes all of out's rows, also past the last sequence."""
    L = contexts
    ctx = L.stub_context()
    plan = make_plan(L, ctx, q=(2, 10), k=(2, 10))
    x, row = _lib.SfeHeads(AT, 128, 64), 256

    def call(out, rows, p=plan):
        return L.sfe_attention_rows(p, _lib.SFE_BF16, x, x, x, None, 0.125, _lib.SfeHeads(out, 128, 64), rows, None)
    passes(L, call(AT + 10 * row, 10))
    passes(L, call(AT + 10 * row, 20))
    passes(L, call(AT - 20 * row, 20))
    refused(L, call(AT - 20 * row, 21), "overlaps")
    refused(L, call(AT + 9 * row, 10), "overlaps")
    refused(L, call(AT + 10 * row, 9), "rows")
    refused(L, call(AT + 10 * row, (1 << 40) + 1), "rows")
    refused(L, call(None, 20), "null out")
    empty, before = make_plan(L, ctx, q=(3, 3), k=(3, 3)), L.stub_calls()
    passes(L, call(AT, 3, empty))
    refused(L, call(None, 4, empty), "null out")
    assert L.stub_calls() == before + 1  # (rows of no sequence are work)
    for p in (plan, empty):
        L.sfe_attention_plan_free(p)
    assert L.stub_destroy(ctx) == 1


# views of one buffer: (row stride, head stride, starts of q and k) in elements of 4 rows, 2 heads, 64 channels
ROWS, HEADS, DIM = 4, 2, 64
LAYOUTS = {"parts of a row": (3 * HEADS * DIM, DIM, 0, HEADS * DIM),
           "parts of a head": (3 * HEADS * DIM, 3 * DIM, 0, DIM),
           "parts of a head, the last before the first": (3 * HEADS * DIM, 3 * DIM, 2 * DIM, 0),
           "heads outermost, parts of a row": (3 * DIM, ROWS * 3 * DIM, 0, DIM),
           "heads outermost, parts of a head": (DIM, 3 * ROWS * DIM, 0, ROWS * DIM),
           "one after the other": (HEADS * DIM, DIM, 0, ROWS * HEADS * DIM)}


def bytes_of(start, row, head, size):
    at = {start + r * row + h * head + d for r in range(ROWS) for h in range(HEADS) for d in range(DIM)}
    return {b for e in at for b in range(e * size, (e + 1) * size)}


def turn_in_place(L, table, q, k):
    return L.sfe_rotary(CTX, ctypes.byref(table), 0, _lib.SFE_BF16, AT - 4096, ROWS, DIM, HEADS, q, q, HEADS, k, k, None)


@pytest.fixture
def table(checks):
    t = _lib.SfeRotaryTable()
    passes(checks, checks.sfe_rotary_init(ctypes.byref(t), DIM, 0, 1e4, 0, 1.0, 1.0, 0.0, 1.0, 1.0))
    return t


@pytest.mark.parametrize("layout", LAYOUTS)
def test_views_of_one_projection(contexts, table, layout):
    """Views that lie between each other without sharing a byte are no overlap, in any order of rows, heads and parts."""
    L = contexts
    row, head, q0, k0 = LAYOUTS[layout]
    q, k = (_lib.SfeHeads(AT + 2 * x, row, head) for x in (q0, k0))
    assert not bytes_of(q0, row, head, 2) & bytes_of(k0, row, head, 2)
    passes(L, turn_in_place(L, table, q, k))
    ctx = L.stub_context()
    plan = make_plan(L, ctx, q=(0, ROWS), k=(0, ROWS))
    passes(L, L.sfe_attention(plan, _lib.SFE_BF16, q, q, q, None, 0.125, k, None))
    L.sfe_attention_plan_free(plan)
    L.stub_destroy(ctx)


def test_views_are_refused_where_they_share_a_byte(contexts, table):
    """For k moved over q by every 16 bytes, the views of each layout: refused whenever bytes are shared."""
    L = contexts
    for row, head, q0, _ in LAYOUTS.values():
        mine = bytes_of(q0, row, head, 2)
        q = _lib.SfeHeads(AT + 2 * q0, row, head)
        for k0 in range(0, 3 * ROWS * HEADS * DIM, 8):
            rc = turn_in_place(L, table, q, _lib.SfeHeads(AT + 2 * k0, row, head))
            if mine & bytes_of(k0, row, head, 2):
                refused(L, rc, "overlaps")


def test_views_of_other_strides(contexts, table):
    """Strides of q and k that differ: a pitch that divides all of them tells them apart or not."""
    L = contexts
    wide, narrow = 6 * DIM, 3 * DIM
    q = _lib.SfeHeads(AT, 2 * wide, wide)
    passes(L, turn_in_place(L, table, q, _lib.SfeHeads(AT + 2 * DIM, 2 * narrow, narrow)))
    refused(L, turn_in_place(L, table, q, _lib.SfeHeads(AT + 2 * (DIM - 8), 2 * narrow, narrow)), "overlaps")
    refused(L, turn_in_place(L, table, q, _lib.SfeHeads(AT + 2 * (wide - 8), 2 * narrow, narrow)), "overlaps")


def test_a_beam_steps_outputs_share_memory_with_nothing(checks):
    """Streams are chosen side by side: an output over part of an input or of another output raced."""
    L, streams, beams, vocab = checks, 2, 3, 10
    place = {"logits": AT, "scores": AT + 1000, "finished": AT + 2000, "out_scores": AT + 3000, "parents": AT + 4000,
             "tokens": AT + 5000, "out_finished": AT + 6000}

    def select(**moved):
        p = {**place, **moved}
        return L.sfe_beam_select(CTX, 0, p["logits"], 12, streams, beams, vocab, p["scores"], p["finished"], 3,
                                 p["out_scores"], p["parents"], p["tokens"], p["out_finished"], None)
    passes(L, select())
    passes(L, select(out_finished=None))
    passes(L, select(out_scores=AT + 1024, parents=AT + 1048, tokens=AT + 1072, out_finished=AT + 2006))
    passes(L, select(scores=AT + 5 * 48 + 40))  # (right behind the last row's 10 logits)
    passes(L, select(out_finished=AT + 2 * 48 + 42))  # (between rows)
    refused(L, select(out_finished=AT + 2 * 48 + 43), "overlaps")
    for out, size in (("out_scores", 24), ("parents", 24), ("tokens", 24), ("out_finished", 6)):
        for other, length in (("logits", 5 * 48 + 40), ("scores", 24), ("finished", 6), ("out_scores", 24), ("parents", 24),
                              ("tokens", 24), ("out_finished", 6)):
            if out == other:
                continue
            step = 1 if out == "out_finished" else 4
            last = (length - 1) // step * step  # the last place that begins within the other
            for at in (0, last, step - size if step < size else 0):
                refused(L, select(**{out: place[other] + at}), "overlap")
            passes(L, select(**{out: place[other] - size}))
            passes(L, select(**{out: (place[other] + length + step - 1) // step * step}))
