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
