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
