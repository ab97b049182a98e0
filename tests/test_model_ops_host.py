"""The model operators' host side without a GPU: the attention's planner, the rotary table, and the
C ABI's refusals (all arguments are checked before any device work)."""
import ctypes
import os
import subprocess
from fractions import Fraction

import pytest

from scriptrs_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "scriptrs_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def plan_driver(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    exe = str(tmp_path_factory.mktemp("attn") / "attn_plan")
    subprocess.run([HIPCC, "-O1", "-g", "-std=c++17", "-x", "hip", "--cuda-host-only", "-Wno-unused-command-line-argument",
                    "-I", os.path.join(ROOT, "include"), "-I", CSRC, os.path.join(ROOT, "tests", "attn_plan_driver.cpp"),
                    os.path.join(CSRC, "sfe_attn_plan.cpp"), "-o", exe], check=True, stderr=subprocess.DEVNULL)
    return exe


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_every_visible_pair_is_in_one_piece(plan_driver, seed):
    r = subprocess.run([plan_driver, str(seed)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "bad 0", r.stdout + r.stderr


def test_rotary_steps():
    """base^(-2p / R) / 2 pi as a fraction of 2^64, to the double's precision."""
    import math
    t = _lib.SfeRotaryTable()
    assert _lib.lib().sfe_rotary_init(ctypes.byref(t), 64, 0, 10_000.0, 0, 1.0, 1.0, 0.0, 1.0, 1.5) == _lib.SFE_OK
    assert (t.rotary_dim, t.layout, t.magnitude) == (64, 0, 1.5)
    for p in range(32):
        want = Fraction(10_000.0 ** (-2 * p / 64) / (2 * math.pi)) * 2 ** 64
        assert abs(t.step[p] - want) <= want * Fraction(1, 2 ** 50) + 1, p
    assert all(t.step[p] == 0 for p in range(32, 128))


def heads(n=1 << 20, row=128, head=64):
    return _lib.SfeHeads(n, row, head)


def refused(rc, part):
    assert rc == _lib.SFE_INVALID_ARG and part in _lib.last_error(), (rc, _lib.last_error())


def test_attention_refusals():
    L = _lib.lib()
    out = ctypes.c_void_p()

    def plan(q=(0, 4), k=(0, 4), h=2, kh=2, d=64, left=-1, right=-1, ctx=None):
        qa, ka = (ctypes.c_int64 * len(q))(*q), (ctypes.c_int64 * len(k))(*k)
        return L.sfe_attention_plan(ctx, qa, ka, len(q) - 1, h, kh, d, left, right, None, ctypes.byref(out))
    refused(plan(), "null context")
    refused(plan(h=3), "multiple of kv_heads")
    refused(plan(h=0), "multiple of kv_heads")
    refused(plan(kh=0), "multiple of kv_heads")
    refused(plan(h=2048), "more than 1024 heads")
    refused(plan(d=60), "head_dim")
    refused(plan(d=136), "head_dim")
    refused(plan(q=(0, -1)), "non-decreasing")
    refused(plan(k=(-2, 4)), "negative")
    refused(plan(q=(0, 1 << 31)), "longer than 2^30")
    refused(plan(q=(0, 1 << 29), h=8), "grouped heads")
    refused(L.sfe_attention_plan(None, None, None, 0, 2, 2, 64, -1, -1, None, ctypes.byref(out)), "null offsets")
    h = heads()
    refused(L.sfe_attention(None, 1, h, h, h, None, 1.0, h, None), "null argument")
    L.sfe_attention_plan_free(None)


def test_rotary_refusals():
    L = _lib.lib()
    t = _lib.SfeRotaryTable()
    init = L.sfe_rotary_init
    refused(init(ctypes.byref(t), 31, 0, 1e4, 0, 1, 1, 0, 1, 1), "rotary_dim")
    refused(init(ctypes.byref(t), 258, 0, 1e4, 0, 1, 1, 0, 1, 1), "rotary_dim")
    refused(init(ctypes.byref(t), 32, 2, 1e4, 0, 1, 1, 0, 1, 1), "layout")
    refused(init(ctypes.byref(t), 32, 0, float("nan"), 0, 1, 1, 0, 1, 1), "base")
    refused(init(ctypes.byref(t), 32, 0, 1e4, 4, 1, 1, 0, 1, 1), "scaling")
    refused(init(ctypes.byref(t), 32, 0, 1e4, 1, 0.5, 1, 0, 1, 1), "factor")
    refused(init(ctypes.byref(t), 32, 0, 1e4, 3, 2, 0, 0, 1, 1), "original_length")
    refused(init(None, 32, 0, 1e4, 0, 1, 1, 0, 1, 1), "null")
    refused(L.sfe_rotary(None, ctypes.byref(t), 0, 0, 1, 4, 32, 1, heads(), heads(), 0, None, None, None), "not initialised")
    assert init(ctypes.byref(t), 32, 0, 1e4, 0, 1, 1, 0, 1, 1) == _lib.SFE_OK
    refused(L.sfe_rotary(None, ctypes.byref(t), 0, 3, 1, 4, 32, 1, heads(), heads(), 0, None, None, None), "dtype")
    refused(L.sfe_rotary(None, ctypes.byref(t), 0, 0, 1, 4, 16, 1, heads(), heads(), 0, None, None, None), "head_dim")
    refused(L.sfe_rotary(None, ctypes.byref(t), 0, 0, 1, -1, 32, 1, heads(), heads(), 0, None, None, None), "rows")
    refused(L.sfe_rotary(None, ctypes.byref(t), 0, 0, 1, 4, 32, 1, heads(), heads(), 0, None, None, None), "null context")


def test_residual_norm_refusals():
    L = _lib.lib()

    def call(**kw):
        a = _lib.SfeResidual()
        a.rows, a.width, a.scale, a.eps = 4, 64, 1.0, 1e-5
        for k, v in kw.items():
            setattr(a, k, v)
        return L.sfe_residual_norm(None, ctypes.byref(a), None)
    refused(L.sfe_residual_norm(None, None, None), "null")
    refused(call(), "null context")
    refused(call(stream_dtype=1, block_dtype=0), "stream_dtype")
    refused(call(block_dtype=7), "dtypes")
    refused(call(width=0), "width")
    refused(call(width=16385), "width")
    refused(call(rows=-1), "rows")
    refused(call(pre=3), "unknown pre norm")
    refused(call(post=1), "post norm without weight")
    refused(call(pre=2, pre_weight=64, pre_bias=64), "no bias")
    refused(call(eps=-1.0), "eps")
    refused(call(scale=float("inf")), "scale")


def test_beam_refusals():
    L = _lib.lib()

    def select(dtype=0, streams=2, beams=4, vocab=10, end=-1, finished=None):
        return L.sfe_beam_select(None, dtype, 64, vocab, streams, beams, vocab, 64, finished, end, 128, 192, 256, 320, None)
    refused(select(), "null context")
    refused(select(dtype=5), "dtype")
    refused(select(streams=-1), "streams")
    refused(select(beams=0), "beams")
    refused(select(beams=33), "beams")
    refused(select(vocab=0), "vocab")
    refused(select(end=10), "end_token")
    refused(select(finished=64), "end_token")
    s = (_lib.SfeBeamState * 1)()
    refused(L.sfe_beam_reorder(None, 64, 2, 4, s, 1, None), "null context")
    refused(L.sfe_beam_reorder(None, 64, 2, 40, s, 1, None), "beams")
    refused(L.sfe_beam_reorder(None, 64, 2, 4, s, -1, None), "negative")


@pytest.mark.parametrize("seed", [1, 2])
def test_planner_without_undefined_behaviour(tmp_path, seed):
    """The planner's host run with every undefined operation a trap, conversions and divisions of doubles included."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "attn_plan")
    subprocess.run([HIPCC, "-O1", "-g", "-std=c++17", "-x", "hip", "--cuda-host-only", "-Wno-unused-command-line-argument",
                    "-Xarch_host", "-fsanitize=undefined,float-cast-overflow,float-divide-by-zero",
                    "-Xarch_host", "-fsanitize-trap=all",
                    "-I", os.path.join(ROOT, "include"), "-I", CSRC, os.path.join(ROOT, "tests", "attn_plan_driver.cpp"),
                    os.path.join(CSRC, "sfe_attn_plan.cpp"), "-o", exe], check=True, stderr=subprocess.DEVNULL)
    r = subprocess.run([exe, str(seed)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "bad 0", (r.returncode, r.stdout + r.stderr)


ROTARY_SCALINGS = {"none": (0, 1.0, 1.0, 0.0, 1.0), "linear": (1, 4.0, 1.0, 0.0, 1.0), "base": (2, 8.0, 1.0, 0.0, 1.0),
                   "parts": (3, 8.0, 4096.0, 1.0, 32.0)}


@pytest.mark.parametrize("scaling", ROTARY_SCALINGS)
@pytest.mark.parametrize("R", [2, 30, 64, 96, 128, 256])
def test_rotary_steps_at_the_farthest_position(R, scaling):
    """A step is off by half a unit of 2^-64 turns for its rounding and by a few roundings of 2^-64 of it: at
    position 2^31 - 1 the angle is off by less than 2^-32 of a turn.  In 60 digits; the inputs are doubles."""
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    kind, factor, length, low, high = ROTARY_SCALINGS[scaling]
    if scaling == "base" and R < 4:
        pytest.skip("scaling the base needs at least 2 pairs")
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    base = 500_000.0
    log_base = Decimal(base).ln() + (Decimal(factor).ln() * R / (R - 2) if scaling == "base" else 0)
    t = _lib.SfeRotaryTable()
    assert _lib.lib().sfe_rotary_init(ctypes.byref(t), R, 0, base, kind, factor, length, low, high, 1.0) == _lib.SFE_OK
    for p in range(R // 2):
        f = (log_base * -2 * p / R).exp()
        if scaling == "linear":
            f /= Decimal(factor)
        if scaling == "parts":
            keep = min(Decimal(1), max(Decimal(0), (Decimal(length) * f / two_pi - Decimal(low)) / Decimal(high - low)))
            f *= (1 - keep) / Decimal(factor) + keep
        want = f / two_pi * 2 ** 64
        assert abs(t.step[p] - want) <= Decimal("0.5") + want / 2 ** 61, p
        assert abs(t.step[p] - want) * (2 ** 31 - 1) < 2 ** 32, p
