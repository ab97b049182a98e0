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
import math

import numpy as np

from . import _lib
from ._lib import SfeBeamState, SfeHeads, SfeResidual, SfeRotaryTable
from .frontend import InvalidModelOutput, ParakeetFeatureExtractor, _check, _ip, _stream_handle

MAX_BEAMS = 32


def _dtype_of(t, what: str) -> int:
    import torch
    code = {torch.float32: _lib.SFE_F32, torch.bfloat16: _lib.SFE_BF16, torch.float16: _lib.SFE_F16}.get(t.dtype)
    if code is None:
        raise InvalidModelOutput(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _on_device(device: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if not getattr(t, "is_cuda", False):
            raise InvalidModelOutput(f"{name} must be a device tensor")
        if t.device.index != device:
            raise InvalidModelOutput(f"{name} is on {t.device}, the operators are on cuda:{device}")


def _heads(t, name: str) -> SfeHeads:
    """A [rows, heads, channels] tensor, channels contiguous."""
    if t.dim() != 3:
        raise InvalidModelOutput(f"{name} must be [rows, heads, channels], got {list(t.shape)}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise InvalidModelOutput(f"{name}: channels must be contiguous")
    return SfeHeads(t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2],
                    t.stride(1) if t.shape[1] > 1 else t.shape[2])


def _same(t, like, name: str) -> None:
    if t.dtype != like.dtype or t.shape != like.shape:
        raise InvalidModelOutput(f"{name} must be {like.dtype} of {list(like.shape)}, got {t.dtype} of {list(t.shape)}")


def _contiguous(t, name: str, dtype, shape) -> int:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise InvalidModelOutput(f"{name} must be a contiguous {dtype} tensor of {list(shape)}, got {t.dtype} of "
                                 f"{list(t.shape)}")
    return t.data_ptr()


def _ref(x):
    return ctypes.byref(x) if x is not None else None


class RotaryTable:
    """Turns a position of each channel pair (``sfe_rotary_table``).

    ``layout``: "half" pairs channel p with p + rotary_dim / 2, "interleaved"
    2p with 2p + 1.  ``scaling`` for long contexts: None, "linear" (positions /
    factor), "base" (base * factor^(R / (R - 2))) or "parts" (pairs that turn at least
    ``high`` times in ``original_length`` positions are kept, those below
    ``low`` divided by ``factor``, the ones between in proportion)."""

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
        _check(_lib.lib().sfe_rotary_init(ctypes.byref(self.c), int(rotary_dim), self.LAYOUTS[layout], float(base),
                                          self.SCALINGS[scaling], float(factor), float(original_length), float(low),
                                          float(high), float(magnitude)))
        self.rotary_dim, self.layout = int(rotary_dim), layout


class AttentionPlan:
    """Division of a batch's sequences into tiles; made by
    ``ModelOps.attention_plan`` and good for every layer over the same lengths."""

    def __init__(self, ops: "ModelOps", handle, total_q: int, total_k: int, heads: int, kv_heads: int, head_dim: int):
        self._ops, self._handle = ops, handle
        self.total_q, self.total_k = total_q, total_k
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim

    def close(self) -> None:
        if self._handle and self._ops._fe._ctx:  # (a closed context has freed it)
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
    ``sfe_ctx`` or shares ``extractor``'s; calls on it are ordered after each other)."""

    def __init__(self, device: int = 0, extractor: ParakeetFeatureExtractor | None = None):
        self._own = extractor is None
        self._fe = extractor or ParakeetFeatureExtractor(device=device)
        self.device = self._fe.device

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
        _check(_lib.lib().sfe_attention_plan(self._fe._handle(), _ip(qo), _ip(ko), qo.size - 1, int(heads), int(kv_heads),
                                             int(head_dim), int(left), int(right), _stream_handle(stream),
                                             ctypes.byref(handle)))
        return AttentionPlan(self, handle, int(qo[-1]), int(ko[-1]), int(heads), int(kv_heads), int(head_dim))

    def attention(self, plan: AttentionPlan, q, k, v, key_mask=None, scale: float | None = None, stream=None, out=None):
        """``softmax(scale q k^T) v`` of each of the plan's sequences:
        ``q`` [queries, heads, head_dim], ``k`` and ``v`` [keys, kv_heads, head_dim] in
        bfloat16 or float16 (views of a joint projection will do), ``key_mask``
        [keys] bool, False hides a key.  Queries that see no key give zeros."""
        import torch
        _on_device(self.device, q=q, k=k, v=v, key_mask=key_mask, out=out)
        if plan._handle is None:
            raise InvalidModelOutput("the plan is closed")
        if plan._ops is not self:
            raise InvalidModelOutput("the plan belongs to another ModelOps")
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise InvalidModelOutput(f"q must be bfloat16 or float16, got {q.dtype}")
        for name, t, n, h in (("q", q, plan.total_q, plan.heads), ("k", k, plan.total_k, plan.kv_heads),
                              ("v", v, plan.total_k, plan.kv_heads)):
            if t.dtype != q.dtype or t.dim() != 3 or t.shape[0] < n or t.shape[1:] != (h, plan.head_dim):
                raise InvalidModelOutput(f"{name} must be {q.dtype} of [{n}, {h}, {plan.head_dim}], got {t.dtype} of "
                                         f"{list(t.shape)}")
        mask = None
        if key_mask is not None:
            if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.dim() != 1 or \
                    key_mask.shape[0] < plan.total_k or not key_mask.is_contiguous():
                raise InvalidModelOutput(f"key_mask must be a contiguous bool tensor of [{plan.total_k}]")
            mask = key_mask.data_ptr()
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _same(out, q, "out")
        if q.shape[0] > plan.total_q:
            out[plan.total_q:].zero_()
        qh, kh, vh, oh = (_heads(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out")))
        _check(_lib.lib().sfe_attention(plan._handle, _dtype_of(q, "q"), ctypes.byref(qh), ctypes.byref(kh),
                                        ctypes.byref(vh), mask,
                                        1.0 / math.sqrt(plan.head_dim) if scale is None else float(scale),
                                        ctypes.byref(oh), _stream_handle(stream)))
        return out

    # -- rotary positions ----------------------------------------------------------
    def rotary(self, table: RotaryTable, positions, q, k=None, inverse: bool = False, inplace: bool = False,
               stream=None):
        """``q`` (and ``k``) [rows, heads, head_dim] turned by ``positions``
        [rows] int32; returns ``(q, k)`` (k None without one).  ``inverse`` turns back."""
        import torch
        _on_device(self.device, positions=positions, q=q, k=k)
        rows, dim = q.shape[0], q.shape[-1]
        pos = _contiguous(positions, "positions", torch.int32, (rows,))
        code = _dtype_of(q, "q")
        if k is not None and (k.dtype != q.dtype or k.dim() != 3 or k.shape[0] != rows or k.shape[2] != dim):
            raise InvalidModelOutput(f"k must be {q.dtype} of [{rows}, heads, {dim}], got {k.dtype} of {list(k.shape)}")
        qo = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = None if k is None else k if inplace else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        qh, qoh = _heads(q, "q"), _heads(qo, "q")
        kh, koh = (None, None) if k is None else (_heads(k, "k"), _heads(ko, "k"))
        _check(_lib.lib().sfe_rotary(self._fe._handle(), ctypes.byref(table.c), 1 if inverse else 0, code, pos, rows,
                                     dim, q.shape[1], ctypes.byref(qh), ctypes.byref(qoh),
                                     0 if k is None else k.shape[1], _ref(kh), _ref(koh), _stream_handle(stream)))
        return qo, ko

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
        import torch
        _on_device(self.device, residual=residual, block=block, gate=gate, post_weight=post_weight, post_bias=post_bias,
                   pre_weight=pre_weight, pre_bias=pre_bias, out=out, norm_out=norm_out)
        if post not in self._NORMS or pre not in self._NORMS:
            raise InvalidModelOutput("norms are None, 'layer' or 'rms'")
        if gate_activation not in (None, "sigmoid"):
            raise InvalidModelOutput(f"unknown gate activation {gate_activation!r}")
        if residual.dim() != 2 or block.shape != residual.shape:
            raise InvalidModelOutput(f"residual and block must be [rows, width], got {list(residual.shape)} and "
                                     f"{list(block.shape)}")
        rows, width = residual.shape
        a = SfeResidual()
        a.stream_dtype, a.block_dtype = _dtype_of(residual, "residual"), _dtype_of(block, "block")
        a.rows, a.width, a.post, a.pre = rows, width, self._NORMS[post], self._NORMS[pre]
        a.gate_sigmoid, a.scale, a.eps = int(gate_activation == "sigmoid"), float(scale), float(eps)

        def put(name, t):
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise InvalidModelOutput(f"{name}: channels must be contiguous")
            setattr(a, name, t.data_ptr())
            setattr(a, name + "_row", t.stride(0) if rows > 1 else width)
        put("residual", residual)
        put("block", block)
        if gate is not None:
            if gate.dtype != block.dtype or gate.shape not in ((width,), residual.shape):
                raise InvalidModelOutput(f"gate must be {block.dtype} of [{width}] or [{rows}, {width}], got {gate.dtype} "
                                         f"of {list(gate.shape)}")
            put("gate", gate.expand(rows, width) if gate.dim() == 1 else gate)
        for name, w in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight),
                        ("pre_bias", pre_bias)):
            if w is not None:
                setattr(a, name, _contiguous(w, name, torch.float32, (width,)))
        x = torch.empty(residual.shape, dtype=residual.dtype, device=residual.device) if out is None else out
        _same(x, residual, "out")
        put("residual_out", x)
        z = None
        if pre is not None:
            z = torch.empty(block.shape, dtype=block.dtype, device=block.device) if norm_out is None else norm_out
            _same(z, block, "norm_out")
            put("norm_out", z)
        _check(_lib.lib().sfe_residual_norm(self._fe._handle(), ctypes.byref(a), _stream_handle(stream)))
        return x, z

    # -- beam search --------------------------------------------------------------------
    def beam_select(self, logits, scores, finished=None, end_token: int = -1, stream=None):
        """A step of beam search: ``logits`` [streams * beams, vocab] (float32, bfloat16
        or float16), ``scores`` [streams, beams] float32, ``finished`` [streams, beams]
        bool.  Returns the best candidates, best first, as ``(scores, parents, tokens,
        finished)`` of [streams, beams] (float32, int32, int32, bool); ties go to
        the lowest (beam, token), a place without a candidate has score -inf and token -1."""
        import torch
        _on_device(self.device, logits=logits, scores=scores, finished=finished)
        if scores.dim() != 2:
            raise InvalidModelOutput(f"scores must be [streams, beams], got {list(scores.shape)}")
        streams, beams = scores.shape
        if logits.dim() != 2 or logits.shape[0] != streams * beams or (logits.shape[1] > 1 and logits.stride(1) != 1):
            raise InvalidModelOutput(f"logits must be [{streams * beams}, vocab] with contiguous rows, got "
                                     f"{list(logits.shape)}")
        code, vocab = _dtype_of(logits, "logits"), logits.shape[1]
        sp = _contiguous(scores, "scores", torch.float32, (streams, beams))
        fp = None
        if finished is not None:
            fp = _contiguous(finished, "finished", torch.bool, (streams, beams))
        new = torch.empty_like(scores)
        picked = torch.empty((2, streams, beams), dtype=torch.int32, device=scores.device)
        ended = torch.empty((streams, beams), dtype=torch.bool, device=scores.device)
        _check(_lib.lib().sfe_beam_select(self._fe._handle(), code, logits.data_ptr(),
                                          logits.stride(0) if logits.shape[0] > 1 else vocab, streams, beams, vocab, sp,
                                          fp, int(end_token), new.data_ptr(), picked[0].data_ptr(),
                                          picked[1].data_ptr(), ended.data_ptr(), _stream_handle(stream)))
        return new, picked[0], picked[1], ended

    def beam_reorder(self, parents, states, dim: int = 0, out=None, stream=None):
        """``states`` (contiguous device tensors whose dimension ``dim`` is streams *
        beams) with every beam's state taken from its parent, in one launch.
        ``out``: tensors to write, ``states`` themselves for in place; returns the list
        written."""
        import torch
        states = list(states)
        out = [torch.empty_like(s) for s in states] if out is None else list(out)
        if len(out) != len(states):
            raise InvalidModelOutput("out must have a tensor for each state")
        _on_device(self.device, parents=parents, **{f"state {i}": s for i, s in enumerate(states)},
                   **{f"out {i}": s for i, s in enumerate(out)})
        if parents.dim() != 2:
            raise InvalidModelOutput(f"parents must be [streams, beams], got {list(parents.shape)}")
        streams, beams = parents.shape
        pp = _contiguous(parents, "parents", torch.int32, (streams, beams))
        table = (SfeBeamState * max(1, len(states)))()
        for i, (s, o) in enumerate(zip(states, out)):
            if not s.is_contiguous() or s.dim() <= dim or s.shape[dim] != streams * beams:
                raise InvalidModelOutput(f"state {i} must be contiguous with {streams * beams} beams in dimension {dim}, "
                                         f"got {list(s.shape)}")
            _same(o, s, f"out {i}")
            if not o.is_contiguous():
                raise InvalidModelOutput(f"out {i} must be contiguous")
            table[i] = SfeBeamState(s.data_ptr(), o.data_ptr(), math.prod(s.shape[:dim]),
                                    math.prod(s.shape[dim + 1:]) * s.element_size())
        _check(_lib.lib().sfe_beam_reorder(self._fe._handle(), pp, streams, beams, table, len(states),
                                           _stream_handle(stream)))
        return out
