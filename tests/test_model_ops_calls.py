"""What ModelOps hands to the library, without a GPU: the library's calls are replaced by ones that record their
arguments, and the tensors are the host's (device -1)."""
import contextlib
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


class Streams:
    """torch's streams replaced: which is current, and which tensors were allocated on or held for which."""

    def __init__(self, monkeypatch, ops):
        self.current, self.allocated, self.held = "main", [], []
        empty_like = ops._empty_like

        def allocate(like, **kw):
            t = empty_like(like, **kw)
            self.allocated.append((self.current, t.data_ptr()))
            return t

        def hold(t, stream):
            self.held.append((stream, t.data_ptr()))
        monkeypatch.setattr(ops, "_empty_like", allocate)
        monkeypatch.setattr(torch, "empty_like", allocate)
        monkeypatch.setattr(torch.Tensor, "record_stream", hold)
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: f"stream {handle}")
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.cuda, "stream", self.use)

    @contextlib.contextmanager
    def use(self, stream):
        before, self.current = self.current, stream
        yield
        self.current = before


def operator_calls(ops):
    """Each operator's (inputs, call); the call returns its outputs."""
    from scriptrs_amd import RotaryTable
    plan = ops.attention_plan([0, 4], [0, 4], 2, 2, 64, stream=0)
    plan._handle = ctypes.c_void_p(2)
    h, mask = [torch.zeros(4, 2, 64, dtype=torch.bfloat16) for _ in range(3)], torch.ones(4, dtype=torch.bool)
    pos, w = torch.zeros(4, dtype=torch.int32), [torch.ones(16) for _ in range(4)]
    x = [torch.zeros(4, 16) for _ in range(3)]
    logits, scores, ended = torch.zeros(4, 9), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.bool)
    parents = torch.zeros(2, 2, dtype=torch.int32)
    norms = dict(post="layer", post_weight=w[0], post_bias=w[1], pre="layer", pre_weight=w[2], pre_bias=w[3])
    yield [*h, mask], lambda s: [ops.attention(plan, *h, key_mask=mask, stream=s)]
    yield [pos, *h[:2]], lambda s: ops.rotary(RotaryTable(64), pos, *h[:2], stream=s)
    yield [*x, *w], lambda s: ops.residual_norm(x[0], x[1], gate=x[2], **norms, stream=s)
    yield [logits, scores, ended], lambda s: ops.beam_select(logits, scores, ended, 3, stream=s)
    yield [parents, *x], lambda s: ops.beam_reorder(parents, x, stream=s)
    plan._handle = None


def test_tensors_of_calls_on_another_stream(ops, monkeypatch):
    """Outputs are of the call's stream's memory, inputs are held for it; on the current stream neither is needed."""
    streams = Streams(monkeypatch, ops)
    for given, call in operator_calls(ops):
        for stream in (None, 0):
            streams.allocated.clear()
            outputs = call(stream)
            assert streams.allocated == [("main", t.data_ptr()) for t in outputs] and not streams.held
        streams.allocated.clear()
        outputs = call(77)
        assert streams.allocated == [("stream 77", t.data_ptr()) for t in outputs]
        assert {("stream 77", t.data_ptr()) for t in given} | {("main", t.data_ptr()) for t in outputs} <= set(streams.held)
        streams.held.clear()


def test_given_outputs_are_held_for_another_stream(ops, monkeypatch):
    streams = Streams(monkeypatch, ops)
    x, y = torch.zeros(4, 16), torch.zeros(4, 16)
    parents, out = torch.zeros(2, 2, dtype=torch.int32), [torch.zeros(4, 16) for _ in range(3)]
    ops.residual_norm(x, y, pre="rms", pre_weight=torch.ones(16), out=out[0], norm_out=out[1], stream=77)
    ops.beam_reorder(parents, [x], out=[out[2]], stream=77)
    assert {("stream 77", t.data_ptr()) for t in out} <= set(streams.held) and not streams.allocated


def test_numbers_past_32_bits_are_refused(ops):
    """ctypes would pass their low 32 bits: another token, table or number of heads."""
    from scriptrs_amd import RotaryTable
    logits, scores = torch.zeros(4, 9), torch.zeros(2, 2)
    far = 1 << 32
    row = torch.empty(1, far + 16, dtype=torch.bfloat16)  # (never touched)
    bad = [lambda: ops.beam_select(logits, scores, end_token=far + 3), lambda: ops.beam_select(logits, scores, end_token=-far),
           lambda: ops.attention_plan([0, 4], [0, 4], far + 2, 2, 64, stream=0),
           lambda: ops.attention_plan([0, 4], [0, 4], 2, far + 2, 64, stream=0),
           lambda: ops.attention_plan([0, 4], [0, 4], 2, 2, far + 64, stream=0),
           lambda: RotaryTable(far + 32), lambda: RotaryTable(64 - far),
           lambda: ops.beam_select(row, scores[:1, :1]), lambda: ops.residual_norm(row, row, out=row),
           lambda: ops.rotary(RotaryTable(16), torch.zeros(1, dtype=torch.int32), row.view(1, 1, -1), inplace=True)]
    for i, f in enumerate(bad):
        with pytest.raises(InvalidModelOutput):
            f()
            raise AssertionError(f"call {i} was not refused")
    assert not ops.recorded


@pytest.mark.parametrize("bound,passed", [(1 << 62, 1 << 62), ((1 << 64) + 5, 1 << 62), (-(1 << 64) + 5, -1), (7, 7), (-1, -1)])
def test_windows_past_64_bits_set_no_bound(ops, bound, passed):
    plan = ops.attention_plan([0, 4], [0, 4], 2, 2, 64, left=bound, right=bound, stream=0)
    assert ops.recorded[-1][1][7:9] == (passed, passed)
    plan._handle = None
