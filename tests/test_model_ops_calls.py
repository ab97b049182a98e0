"""What ModelOps hands to the library, without a GPU: the library's calls are replaced by ones that record their
arguments, and the tensors are the host's (device -1)."""
import ctypes

import pytest
import torch

from scriptrs_amd import InvalidModelOutput, ModelOps, _lib


class Extractor:
    """Stands in for the feature extractor: a context that is never looked into."""
    device = -1

    def __init__(self):
        self._ctx = ctypes.c_void_p(1)

    def _handle(self):
        return self._ctx

    def close(self):
        self._ctx = ctypes.c_void_p()


class Library:
    """Records the operators' calls; the rest is the library's own."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name in ("sfe_rotary_init", "sfe_last_error"):
            return getattr(REAL, name)

        def call(*args):
            self.calls.append((name, args))
            return _lib.SFE_OK
        return call


REAL = _lib.lib()


@pytest.fixture
def ops(monkeypatch):
    library = Library()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    m = ModelOps(extractor=Extractor())
    m._stream_of = lambda device: 0
    m.recorded = library.calls
    return m


def states_of(ops):
    name, (_, _, streams, beams, table, n, _) = ops.recorded[-1]
    assert name == "sfe_beam_reorder"
    return [(s.outer, streams * beams, s.inner_bytes) for s in table[:n]]


@pytest.mark.parametrize("shape,dim", [((3, 8), 1), ((3, 8), -1), ((8, 5), 0), ((8, 5), -2), ((2, 8, 7), 1),
                                       ((2, 8, 7), -2), ((8,), -1), ((8,), 0), ((8, 8, 8), -1)])
def test_reordered_states_are_the_tensors(ops, shape, dim):
    """outer x beams x inner is the tensor, with dimensions counted from either end."""
    state = torch.zeros(shape)
    parents = torch.zeros(2, 4, dtype=torch.int32)
    ops.beam_reorder(parents, [state], dim=dim)
    (outer, rows, inner), = states_of(ops)
    at = dim % len(shape)
    assert (outer, rows, inner) == (torch.Size(shape[:at]).numel(), 8, 4 * torch.Size(shape[at + 1:]).numel())
    assert outer * rows * inner == state.numel() * state.element_size()


@pytest.mark.parametrize("dim", [2, -3, 99, -99])
def test_dimensions_that_a_state_does_not_have_are_refused(ops, dim):
    with pytest.raises(InvalidModelOutput, match="dimension"):
        ops.beam_reorder(torch.zeros(2, 4, dtype=torch.int32), [torch.zeros(8, 8)], dim=dim)
    assert not ops.recorded


@pytest.mark.parametrize("order", ["plan first", "context first", "context reopened"])
def test_a_plan_is_freed_once_whatever_its_context(ops, order):
    plan = ops.attention_plan([0, 4], [0, 4], 2, 2, 64, stream=0)
    plan._handle = ctypes.c_void_p(2)
    if order != "plan first":
        ops._fe.close()
    if order == "context reopened":
        ops._fe._ctx = ctypes.c_void_p(3)
    plan.close()
    plan.close()
    freed = [args for name, args in ops.recorded if name == "sfe_attention_plan_free"]
    assert len(freed) == 1 and freed[0][0].value == 2


def test_calls_without_a_stream_take_their_devices(ops):
    """The current stream of the operators' device, which need not be torch's current device."""
    ops._stream_of = lambda device: 1000 + device
    plan = ops.attention_plan([0, 4], [0, 4], 2, 2, 64)
    plan._handle = ctypes.c_void_p(2)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    ops.attention(plan, x, x, x)
    assert {name: args[9 if name == "sfe_attention_plan" else 8] for name, args in ops.recorded} == {
        "sfe_attention_plan": 999, "sfe_attention": 999}
    plan._handle = None


@pytest.mark.parametrize("offsets,rows,name", [([0, 4], 4, "sfe_attention"), ([0, 4], 6, "sfe_attention_rows"),
                                               ([1, 4], 4, "sfe_attention_rows"), ([3], 5, "sfe_attention_rows")])
def test_rows_of_no_sequence_are_part_of_the_call(ops, offsets, rows, name):
    """They are zeroed by the call itself, in the context's order; nothing is queued behind it."""
    plan = ops.attention_plan(offsets, offsets, 2, 2, 64, stream=0)
    plan._handle = ctypes.c_void_p(2)
    q, out = torch.zeros(rows, 2, 64, dtype=torch.bfloat16), torch.ones(rows, 2, 64, dtype=torch.bfloat16)
    ops.attention(plan, q, q, q, out=out, stream=0)
    assert [n for n, _ in ops.recorded] == ["sfe_attention_plan", name] and bool((out == 1).all())
    if name == "sfe_attention_rows":
        assert ops.recorded[-1][1][8] == rows
    plan._handle = None
