"""Operators of the models behind the features, on the GPU.

The features of a ragged batch go through an encoder and a decoder that
searches for the transcript (closed bundles in the reference, src/model.rs).
``ModelOps`` has the operators that such a model is built from beside plain
matrix products: attention over packed sequences with grouped heads, rotary
positions, the norms around a block with its gate and residual scale, and a
step of beam search with its states' reordering.  All of them run in
``libscriptrs_fe.so``; arguments are checked before any device work, and a
refused call raises ``InvalidModelOutput``.
"""
from __future__ import annotations

import ctypes
import functools
import math

import numpy as np

from . import _lib
from ._lib import SfeBeamState, SfeHeads, SfeResidual, SfeRotaryTable
from .frontend import InvalidModelOutput, ParakeetFeatureExtractor, _check, _ip, _stream_handle

MAX_BEAMS = 32
MAX_INT32 = (1 << 31) - 1  # (sizes are passed in 32 bits)

_DTYPES: dict = {}  # torch dtype -> sfe_dtype, filled by the first ModelOps (torch is imported lazily)


def _dtype_of(t, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise InvalidModelOutput(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _wrong_device(name: str, t, device: int):
    if not getattr(t, "is_cuda", False):
        raise InvalidModelOutput(f"{name} must be a device tensor")
    raise InvalidModelOutput(f"{name} is on {t.device}, the operators are on cuda:{device}")


def _heads(t, name: str, shape, out):
    """Writes a [rows, heads, channels] tensor, channels contiguous, into an sfe_heads."""
    rows, heads, dim = shape
    row, head, channel = t.stride()
    if channel != 1 and dim > 1:
        raise InvalidModelOutput(f"{name}: channels must be contiguous")
    out.data = t.data_ptr()
    out.row_stride = row if rows > 1 else heads * dim
    out.head_stride = head if heads > 1 else dim


def _same(t, like, name: str) -> None:
    if t.dtype != like.dtype or t.shape != like.shape:
        raise InvalidModelOutput(f"{name} must be {like.dtype} of {list(like.shape)}, got {t.dtype} of {list(t.shape)}")


def _int32(value, name: str) -> int:
    """An argument that is passed in 32 bits (ctypes would drop the bits above)."""
    value = int(value)
    if not -(1 << 31) <= value < 1 << 31:
        raise InvalidModelOutput(f"{name} does not fit 32 bits: {value}")
    return value


def _contiguous(t, name: str, dtype, shape) -> int:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise InvalidModelOutput(f"{name} must be a contiguous {dtype} tensor of {list(shape)}, got {t.dtype} of "
                                 f"{list(t.shape)}")
    return t.data_ptr()


class RotaryTable:
    """Turns a position of each channel pair (``sfe_rotary_table``).

    ``layout``: "half" pairs channel p with p + rotary_dim / 2, "interleaved"
    2p with 2p + 1.  ``scaling`` for long contexts: None, "linear" (positions /
    factor), "base" (base * factor^(R / (R - 2))) or "parts" (pairs that turn at least
    ``high`` times in ``original_length`` positions are kept, those below
    ``low`` divided by ``factor``, the ones between in proportion to their turns, not to
    their number p: tables that ramp over p are others)."""

    LAYOUTS = {"half": 0, "interleaved": 1}
    SCALINGS = {None: 0, "none": 0, "linear": 1, "base": 2, "parts": 3}

    def __init__(self, rotary_dim: int, layout: str = "half", base: float = 10_000.0, scaling: str | None = None,
                 factor: float = 1.0, original_length: float = 1.0, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 1.0):
        if layout not in self.LAYOUTS:
            raise InvalidModelOutput(f"unknown rotary layout {layout!r}")
        if scaling not in self.SCALINGS:
            raise InvalidModelOutput(f"unknown rotary scaling {scaling!r}")
        self.c = SfeRotaryTable()
        _check(_lib.lib().sfe_rotary_init(ctypes.byref(self.c), _int32(rotary_dim, "rotary_dim"), self.LAYOUTS[layout], float(base),
                                          self.SCALINGS[scaling], float(factor), float(original_length), float(low),
                                          float(high), float(magnitude)))
        self.rotary_dim, self.layout = int(rotary_dim), layout
        self.p = ctypes.byref(self.c)


class AttentionPlan:
    """Division of a batch's sequences into tiles; made by
    ``ModelOps.attention_plan`` and good for every layer over the same lengths, until its context (the
    ``ModelOps`` or the extractor that it shares) is closed."""

    def __init__(self, ops: "ModelOps", handle, first_q: int, total_q: int, total_k: int, heads: int, kv_heads: int,
                 head_dim: int):
        self._ops, self._handle = ops, handle
        self.first_q, self.total_q, self.total_k = first_q, total_q, total_k
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.scale = 1.0 / math.sqrt(head_dim)

    def close(self) -> None:
        if self._handle:
            _lib.lib().sfe_attention_plan_free(self._handle)
        self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class ModelOps:
    """The operators on one device.

    One instance per host thread, like the feature extractor (it owns an
    ``sfe_ctx`` or shares ``extractor``'s; calls on it are ordered after each other).
    ``stream``: a call's stream (torch's, or its handle), the current one without; its inputs have to be ready there, and
    a stream given by its handle has to outlive the tensors of its calls (their memory is held for it)."""

    def __init__(self, device: int = 0, extractor: ParakeetFeatureExtractor | None = None):
        import torch
        self._torch, self._f32 = torch, torch.float32
        _DTYPES.update({torch.float32: _lib.SFE_F32, torch.bfloat16: _lib.SFE_BF16, torch.float16: _lib.SFE_F16})
        # (0.6 us less than new_empty)
        self._empty_like = functools.partial(torch.empty_like, memory_format=torch.contiguous_format)
        self._own = extractor is None
        self._fe = extractor or ParakeetFeatureExtractor(device=device)
        self.device = self._fe.device
        self._lib = _lib.lib()
        self._stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        # argument structs, filled for each call (calls come from one host thread)
        self._h = [SfeHeads() for _ in range(4)]
        self._hp = [ctypes.byref(h) for h in self._h]
        self._residual = SfeResidual()
        self._residual_p = ctypes.byref(self._residual)
        self._states = (SfeBeamState * 8)()

    def _stream(self, stream) -> int | None:
        if stream is None:
            if self._stream_of is not None:
                return self._stream_of(self.device)
            stream = self._torch.cuda.current_stream(self.device)
        return _stream_handle(stream)

    def _other(self, stream):
        """The call's stream as torch's, where it is not the current one."""
        if stream is None:
            return None
        torch, handle = self._torch, _stream_handle(stream).value or 0
        if handle == (self._stream(None) or 0):
            return None
        if isinstance(stream, torch.cuda.Stream):
            return stream
        return torch.cuda.ExternalStream(handle, device=self.device) if handle else torch.cuda.default_stream(self.device)

    def _new(self, other, like, dtype=None):
        """An output, of the memory of the stream that writes it (the current stream's may have just been freed and
        still be in use there), held for the current stream too, on which the caller may read it later."""
        if other is None:
            return self._empty_like(like) if dtype is None else self._empty_like(like, dtype=dtype)
        with self._torch.cuda.stream(other):
            t = self._empty_like(like, dtype=dtype or like.dtype)
        t.record_stream(self._torch.cuda.current_stream(self.device))
        return t

    @staticmethod
    def _held(other, *tensors) -> None:
        """Given tensors keep their memory until the call's stream is done with them, freed meanwhile or not."""
        for t in tensors:
            if t is not None:
                t.record_stream(other)

    def close(self) -> None:
        if self._own:
            self._fe.close()

    # -- attention ---------------------------------------------------------------
    def attention_plan(self, q_offsets, k_offsets, heads: int, kv_heads: int, head_dim: int, left: int = -1,
                       right: int = -1, stream=None) -> AttentionPlan:
        """Plan for sequences ``q_offsets[s]:q_offsets[s + 1]`` of queries over
        ``k_offsets[s]:k_offsets[s + 1]`` of keys.  Queries and keys are aligned at
        their ends; ``left`` / ``right`` limit the keys before / after a query's own
        place (-1: no limit; causal: right=0)."""
        qo, ko = (np.ascontiguousarray(o, np.int64).reshape(-1) for o in (q_offsets, k_offsets))
        if qo.size == 0 or qo.size != ko.size:
            raise InvalidModelOutput("q_offsets and k_offsets must have one entry more than there are sequences")
        handle = ctypes.c_void_p()
        heads, kv_heads, head_dim = _int32(heads, "heads"), _int32(kv_heads, "kv_heads"), _int32(head_dim, "head_dim")
        left, right = (min(max(int(bound), -1), 1 << 62) for bound in (left, right))
        _check(_lib.lib().sfe_attention_plan(self._fe._handle(), _ip(qo), _ip(ko), _int32(qo.size - 1, "sequences"), heads,
                                             kv_heads, head_dim, left, right, self._stream(stream), ctypes.byref(handle)))
        return AttentionPlan(self, handle, int(qo[0]), int(qo[-1]), int(ko[-1]), heads, kv_heads, head_dim)

    def attention(self, plan: AttentionPlan, q, k, v, key_mask=None, scale: float | None = None, stream=None, out=None):
        """``softmax(scale q k^T) v`` of each of the plan's sequences:
        ``q`` [queries, heads, head_dim], ``k`` and ``v`` [keys, kv_heads, head_dim] in
        bfloat16 or float16 (views of a joint projection will do), ``key_mask``
        [keys] bool, False hides a key.  Queries that see no key give zeros, and so do rows
        before the first sequence and past the last."""
        handle = plan._handle
        if handle is None:
            raise InvalidModelOutput("the plan is closed")
        if plan._ops is not self:
            raise InvalidModelOutput("the plan belongs to another ModelOps")
        dtype, device = q.dtype, self.device
        code = _dtype_of(q, "q")
        if code == _lib.SFE_F32:
            raise InvalidModelOutput(f"q must be bfloat16 or float16, got {dtype}")
        hq, hk, hv, ho = self._h
        tail_q, tail_k = (plan.heads, plan.head_dim), (plan.kv_heads, plan.head_dim)
        for name, t, n, tail, h in (("q", q, plan.total_q, tail_q, hq), ("k", k, plan.total_k, tail_k, hk),
                                    ("v", v, plan.total_k, tail_k, hv)):
            if t.get_device() != device:
                _wrong_device(name, t, device)
            shape = t.shape
            if t.dtype != dtype or len(shape) != 3 or shape[0] < n or shape[1:] != tail:
                raise InvalidModelOutput(f"{name} must be {dtype} of [{n}, {tail[0]}, {tail[1]}], got {t.dtype} of "
                                         f"{list(shape)}")
            _heads(t, name, shape, h)
        mask = None
        if key_mask is not None:
            torch = self._torch
            if key_mask.get_device() != device:
                _wrong_device("key_mask", key_mask, device)
            if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.dim() != 1 or \
                    key_mask.shape[0] < plan.total_k or not key_mask.is_contiguous():
                raise InvalidModelOutput(f"key_mask must be a contiguous bool tensor of [{plan.total_k}]")
            mask = key_mask.data_ptr()
        other = None if stream is None else self._other(stream)
        if other is not None:
            self._held(other, q, k, v, key_mask, out)
        if out is None:
            out = self._empty_like(q) if other is None else self._new(other, q)
            ho.data, ho.row_stride, ho.head_stride = out.data_ptr(), plan.heads * plan.head_dim, plan.head_dim
        else:
            _same(out, q, "out")
            if out.get_device() != device:
                _wrong_device("out", out, device)
            _heads(out, "out", q.shape, ho)
        pq, pk, pv, po = self._hp
        if scale is None:
            scale = plan.scale
        if plan.first_q or q.shape[0] > plan.total_q:  # rows of no sequence
            rc = self._lib.sfe_attention_rows(handle, code, pq, pk, pv, mask, scale, po, q.shape[0], self._stream(stream))
        else:
            rc = self._lib.sfe_attention(handle, code, pq, pk, pv, mask, scale, po, self._stream(stream))
        if rc:
            _check(rc)
        return out

    # -- rotary positions ----------------------------------------------------------
    def rotary(self, table: RotaryTable, positions, q, k=None, inverse: bool = False, inplace: bool = False,
               stream=None):
        """``q`` (and ``k``) [rows, heads, head_dim] turned by ``positions``
        [rows] int32; returns ``(q, k)`` (k None without one).  ``inverse`` turns back."""
        torch = self._torch
        device, code, shape = self.device, _dtype_of(q, "q"), q.shape
        if len(shape) != 3:
            raise InvalidModelOutput(f"q must be [rows, heads, channels], got {list(shape)}")
        rows, heads, dim = shape
        if heads > MAX_INT32 or dim > MAX_INT32:
            raise InvalidModelOutput("heads and channels must be below 2^31")
        for name, t in (("positions", positions), ("q", q)):
            if t.get_device() != device:
                _wrong_device(name, t, device)
        pos = _contiguous(positions, "positions", torch.int32, (rows,))
        hq, hqo, hk, hko = self._h
        _heads(q, "q", shape, hq)
        other = None if stream is None else self._other(stream)
        if other is not None:
            self._held(other, positions, q, k)
        q_out = q
        if not inplace:
            q_out = self._empty_like(q) if other is None else self._new(other, q)
            hqo.data, hqo.row_stride, hqo.head_stride = q_out.data_ptr(), heads * dim, dim
        k_out, kv_heads = None, 0
        if k is not None:
            if k.get_device() != device:
                _wrong_device("k", k, device)
            shape = k.shape
            if k.dtype != q.dtype or len(shape) != 3 or shape[0] != rows or shape[2] != dim or shape[1] > MAX_INT32:
                raise InvalidModelOutput(f"k must be {q.dtype} of [{rows}, heads, {dim}], got {k.dtype} of {list(shape)}")
            kv_heads = shape[1]
            _heads(k, "k", shape, hk)
            k_out = k
            if not inplace:
                k_out = self._empty_like(k) if other is None else self._new(other, k)
                hko.data, hko.row_stride, hko.head_stride = k_out.data_ptr(), kv_heads * dim, dim
        pq, pqo, pk, pko = self._hp
        if inplace:
            pqo, pko = pq, pk
        rc = self._lib.sfe_rotary(self._fe._handle(), table.p, 1 if inverse else 0, code, pos, rows, dim, heads, pq, pqo,
                                  kv_heads, pk, pko, self._stream(stream))
        if rc:
            _check(rc)
        return q_out, k_out

    # -- norms around a block ---------------------------------------------------------
    _NORMS = {None: 0, "layer": 1, "rms": 2}

    def residual_norm(self, residual, block, scale: float = 1.0, gate=None, gate_activation: str | None = None,
                      post: str | None = None, post_weight=None, post_bias=None, pre: str | None = None,
                      pre_weight=None, pre_bias=None, eps: float = 1e-5, out=None, norm_out=None, stream=None):
        """``x = residual + scale * gate * N_post(block)`` and ``N_pre(x)``.

        ``residual`` [rows, width] in float32 or ``block``'s dtype; ``gate`` [width]
        or [rows, width], through a sigmoid if ``gate_activation`` is "sigmoid"; norms None,
        "layer" or "rms" with float32 weights (and biases) [width].  Returns
        ``(x, norm)``; norm is None without ``pre``.  ``out`` may be ``residual``
        and ``norm_out`` may be ``block``."""
        if post not in self._NORMS or pre not in self._NORMS:
            raise InvalidModelOutput("norms are None, 'layer' or 'rms'")
        if gate_activation is not None and gate_activation != "sigmoid":
            raise InvalidModelOutput(f"unknown gate activation {gate_activation!r}")
        device, shape = self.device, residual.shape
        if len(shape) != 2 or block.shape != shape:
            raise InvalidModelOutput(f"residual and block must be [rows, width], got {list(shape)} and "
                                     f"{list(block.shape)}")
        rows, width = shape
        if width > MAX_INT32:
            raise InvalidModelOutput(f"width {width} does not fit 32 bits")
        a = self._residual
        a.stream_dtype, a.block_dtype = _dtype_of(residual, "residual"), _dtype_of(block, "block")
        a.rows, a.width, a.post, a.pre = rows, width, self._NORMS[post], self._NORMS[pre]
        a.gate_sigmoid, a.scale, a.eps = 0 if gate_activation is None else 1, scale, eps

        def rows_of(name, t):
            if t.get_device() != device:
                _wrong_device(name, t, device)
            row, channel = t.stride()
            if channel != 1 and width > 1:
                raise InvalidModelOutput(f"{name}: channels must be contiguous")
            return t.data_ptr(), row if rows > 1 else width
        a.residual, a.residual_row = rows_of("residual", residual)
        a.block, a.block_row = rows_of("block", block)
        a.gate = None
        if gate is not None:
            if gate.dtype != block.dtype or gate.shape != (width,) and gate.shape != shape:
                raise InvalidModelOutput(f"gate must be {block.dtype} of [{width}] or [{rows}, {width}], got {gate.dtype} "
                                         f"of {list(gate.shape)}")
            a.gate, a.gate_row = rows_of("gate", gate if gate.dim() == 2 else gate.expand(rows, width))
        a.post_weight = None if post_weight is None else self._weight("post_weight", post_weight, width)
        a.post_bias = None if post_bias is None else self._weight("post_bias", post_bias, width)
        a.pre_weight = None if pre_weight is None else self._weight("pre_weight", pre_weight, width)
        a.pre_bias = None if pre_bias is None else self._weight("pre_bias", pre_bias, width)
        other = None if stream is None else self._other(stream)
        if other is not None:
            self._held(other, residual, block, gate, post_weight, post_bias, pre_weight, pre_bias, out, norm_out)
        if out is None:
            out = self._empty_like(residual) if other is None else self._new(other, residual)
            a.residual_out, a.residual_out_row = out.data_ptr(), width
        else:
            _same(out, residual, "out")
            a.residual_out, a.residual_out_row = rows_of("out", out)
        if pre is None:
            norm_out = a.norm_out = None
        elif norm_out is None:
            norm_out = self._empty_like(block) if other is None else self._new(other, block)
            a.norm_out, a.norm_out_row = norm_out.data_ptr(), width
        else:
            _same(norm_out, block, "norm_out")
            a.norm_out, a.norm_out_row = rows_of("norm_out", norm_out)
        rc = self._lib.sfe_residual_norm(self._fe._handle(), self._residual_p, self._stream(stream))
        if rc:
            _check(rc)
        return out, norm_out

    def _weight(self, name: str, w, width: int) -> int:
        if w.get_device() != self.device:
            _wrong_device(name, w, self.device)
        if w.dtype != self._f32 or w.shape != (width,) or not w.is_contiguous():
            raise InvalidModelOutput(f"{name} must be a contiguous float32 tensor of [{width}], got {w.dtype} of "
                                     f"{list(w.shape)}")
        return w.data_ptr()

    # -- beam search --------------------------------------------------------------------
    def beam_select(self, logits, scores, finished=None, end_token: int = -1, stream=None):
        """A step of beam search: ``logits`` [streams * beams, vocab] (float32, bfloat16
        or float16), ``scores`` [streams, beams] float32, ``finished`` [streams, beams]
        bool.  Returns the best candidates, best first, as ``(scores, parents, tokens,
        finished)`` of [streams, beams] (float32, int32, int32, bool); ties go to
        the lowest (beam, token), a place without a candidate has score -inf and token -1."""
        torch = self._torch
        device, shape = self.device, scores.shape
        if len(shape) != 2:
            raise InvalidModelOutput(f"scores must be [streams, beams], got {list(shape)}")
        streams, beams = shape
        if logits.dim() != 2 or logits.shape[0] != streams * beams or (logits.stride(1) != 1 and logits.shape[1] > 1):
            raise InvalidModelOutput(f"logits must be [{streams * beams}, vocab] with contiguous rows, got "
                                     f"{list(logits.shape)}")
        for name, t in (("logits", logits), ("scores", scores)):
            if t.get_device() != device:
                _wrong_device(name, t, device)
        code, vocab = _dtype_of(logits, "logits"), logits.shape[1]
        if not -1 <= end_token < vocab <= MAX_INT32 or streams > MAX_INT32 or beams > MAX_INT32:
            raise InvalidModelOutput(f"end_token must be a token, or -1, and sizes below 2^31: got {end_token}, {streams} x "
                                     f"{beams} beams of {vocab}")
        sp, fp = _contiguous(scores, "scores", torch.float32, shape), None
        if finished is not None:
            if finished.get_device() != device:
                _wrong_device("finished", finished, device)
            fp = _contiguous(finished, "finished", torch.bool, shape)
        other = None if stream is None else self._other(stream)
        if other is not None:
            self._held(other, logits, scores, finished)
        new = self._new(other, scores)
        parents, tokens = self._new(other, scores, torch.int32), self._new(other, scores, torch.int32)
        ended = self._new(other, scores, torch.bool)
        rc = self._lib.sfe_beam_select(self._fe._handle(), code, logits.data_ptr(), logits.stride(0), streams, beams,
                                       vocab, sp, fp, end_token, new.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                                       ended.data_ptr(), self._stream(stream))
        if rc:
            _check(rc)
        return new, parents, tokens, ended

    def beam_reorder(self, parents, states, dim: int = 0, out=None, stream=None):
        """``states`` (contiguous device tensors whose dimension ``dim``, from the end if negative, is
        streams * beams) with every beam's state taken from its parent, in one launch.
        ``out``: tensors to write, ``states`` themselves for in place (an output may share memory with
        no other tensor); returns the list written."""
        torch = self._torch
        states = list(states)
        given = None if out is None else list(out)
        if given is not None and len(given) != len(states):
            raise InvalidModelOutput("out must have a tensor for each state")
        if parents.get_device() != self.device:
            _wrong_device("parents", parents, self.device)
        shape = parents.shape
        if len(shape) != 2 or max(shape) > MAX_INT32:
            raise InvalidModelOutput(f"parents must be [streams, beams], got {list(shape)}")
        streams, beams = shape
        pp = _contiguous(parents, "parents", torch.int32, shape)
        n, out = len(states), []
        other = None if stream is None else self._other(stream)
        if other is not None:
            self._held(other, parents)
        table = self._states if n <= len(self._states) else (SfeBeamState * n)()
        for i, s in enumerate(states):
            if s.get_device() != self.device:
                _wrong_device(f"state {i}", s, self.device)
            full = s.shape
            at = dim + len(full) if dim < 0 else dim
            if not s.is_contiguous() or not 0 <= at < len(full) or full[at] != streams * beams:
                raise InvalidModelOutput(f"state {i} must be contiguous with {streams * beams} beams in dimension {dim}, "
                                         f"got {list(full)}")
            if given is None:
                o = self._new(other, s)
            else:
                o = given[i]
                if o.get_device() != self.device:
                    _wrong_device(f"out {i}", o, self.device)
                _same(o, s, f"out {i}")
                if not o.is_contiguous():
                    raise InvalidModelOutput(f"out {i} must be contiguous")
            out.append(o)
            if other is not None:
                self._held(other, s, o)
            row = table[i]
            row.in_, row.out = s.data_ptr(), o.data_ptr()
            row.outer, row.inner_bytes = math.prod(full[:at]), math.prod(full[at + 1:]) * s.element_size()
        rc = self._lib.sfe_beam_reorder(self._fe._handle(), pp, streams, beams, table, n, self._stream(stream))
        if rc:
            _check(rc)
        return out
