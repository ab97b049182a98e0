"""Refusals of a decoder's step over a paged cache at the ends of their ranges, without a GPU (built as in
test_decode_checks.py)."""
import ctypes

from test_decode_checks import AT, cache, checks, ctx, heads, make, passes, refused, tokens  # noqa: F401


def test_attention_of_no_new_tokens_keeps_what_its_rows_would_lie_over(checks, ctx):  # noqa: F811
    """Rows of no sequence are zeroed also where the plan has none: not over the cache, the table or the lengths."""
    L = checks
    plan = make(L, ctx, (0, 0, 0))[1]

    def attend(out, t=None, tree=None):
        return L.sfe_cache_attention(plan, ctypes.byref(cache()), ctypes.byref(t or tokens()), 1, heads(2 * AT, 256), tree, 0.125, out, 3, None)
    passes(L, attend(heads(3 * AT, 256)))
    passes(L, attend(heads(2 * AT, 256)))  # (q, of which nothing is read)
    passes(L, attend(heads(3 * AT, 256), t=tokens(0, 0, 0, 0)))
    refused(L, attend(heads(AT, 256)), "out overlaps the cache")
    refused(L, attend(heads(AT - 512, 256)), "out overlaps the cache")
    refused(L, attend(heads(AT - 8192, 256)), "out overlaps page_table")
    refused(L, attend(heads(AT - 4096 - 16, 256)), "out overlaps lengths")
    L.sfe_cache_plan_free(plan)


def test_repetitions_without_a_reciprocal(checks):  # noqa: F811
    """Below f32's normal numbers a reciprocal is infinite, and with it every quotient of 16-bit logits."""
    import struct
    from scriptrs_amd import _lib
    least = 2.0 ** -126
    below = struct.unpack("f", struct.pack("I", 0x007fffff))[0]

    def call(repetition, each=None, history=AT * 3):
        a = _lib.SfeLogits(dtype=1, rows=4, vocab=100, history_most=8, logits=AT, out=AT * 2, logits_row=100, out_row=100, history=history,
                           history_row=8, repetition=repetition, repetitions=each)
        return checks.sfe_adjust_logits(ctypes.c_void_p(1), ctypes.byref(a), None)
    passes(checks, call(least))
    refused(checks, call(below), "repetition")
    refused(checks, call(2.0 ** -149), "repetition")
    passes(checks, call(below, each=AT * 8))  # (the rows' own count)
