"""Paged key-value cache: what a serving loop writes into it and reads from it.

The cache is two tensors of pages, ``k_cache`` and ``v_cache`` [num_blocks, H_k, block, D] (bf16,
f16, f32 or fp8 e4m3), a ``block_table`` int32 [B, W] from a sequence's logical pages to pages, and
``context_lens`` int32 [B] (other integers are converted, by a kernel or two a call). Per decode step and
layer:

    q = paged.paged_append(k, v, k_cache, v_cache, block_table, context_lens, q=q, cos=cos, sin=sin)
    out = paged.paged_decode_attn(q, k_cache, v_cache, block_table, context_lens, D ** -0.5)

or, with page summaries (``new_block_summary``) kept by the append, attention over the pages whose
8-bit key minima and maxima score highest:

    out = paged.paged_sparse_decode_attn(q, k_cache, v_cache, summary, summary_scale, block_table,
                                         context_lens, 64, D ** -0.5)

All calls run on the current stream, allocate their outputs and scratch from torch's caching
allocator, read lengths and tables on the device only, and can be captured in CUDA graphs. The
reference pages its PQ caches only; there is no counterpart of these there. There is no CPU path.
"""
import torch

from . import _native as N


def _pair(a, b, names):
    if (a is None) != (b is None):
        raise ValueError(f"{names} go together")


def new_block_summary(k_cache):
    """Zeroed (summary int8 [num_blocks, H_k, 2, D], summary_scale f32 [num_blocks, H_k]) for a cache."""
    nb, hk, _, d = k_cache.shape
    return (torch.zeros(nb, hk, 2, d, dtype=torch.int8, device=k_cache.device),
            torch.zeros(nb, hk, dtype=torch.float32, device=k_cache.device))


def paged_append(k, v, k_cache, v_cache, block_table, context_lens, *, q=None, cos=None, sin=None, interleaved=False,
                 cu_seqlens=None, k_scale=1.0, v_scale=1.0, summary=None, summary_scale=None):
    """Write new tokens' keys and values into their pages in place, keys rotated by their position;
    returns the rotated queries (None without q).

    k, v [T, H_k, D] and q [T, H_q, D] (bf16 / f16 / f32, any strides: views of one projection's
    output will do). ``context_lens`` counts the new tokens already. ``cu_seqlens`` int32 [B+1] gives
    each sequence's run of packed tokens (None: one token for each sequence). cos, sin f32
    [positions, r/2] rotate the first r channels by pairs (i, i + r/2), or (2i, 2i+1) if
    ``interleaved``; None leaves keys and queries as they are. An fp8 cache holds x / k_scale and
    x / v_scale, cut to the type's range. With ``summary`` and ``summary_scale`` the summaries of the
    touched pages are renewed. Tokens without a place (past cu_seqlens[-1], a sequence of length 0,
    past the block table or past the rows of cos, or an entry that names no page) are not written;
    their query rows come back as zeros.
    """
    _pair(cos, sin, "cos and sin")
    _pair(summary, summary_scale, "summary and summary_scale")
    rc, q_out = N.glue().paged_append(k, v, k_cache, v_cache, block_table, context_lens, q, cos, sin, interleaved,
                                      cu_seqlens, k_scale, v_scale, summary, summary_scale)
    if rc:
        N.check(rc, "bd_paged_append")
    return q_out


def paged_block_summary(k_cache, block_table, context_lens, summary, summary_scale, *, k_scale=1.0):
    """Renew the summaries of every page that holds tokens of the sequences, in place.

    Per page and KV head, over the page's tokens: channelwise minimum and maximum of k_scale * key as
    int8 codes rint(x / s), s = max|x| / 127. Keys that are NaN do not count (a channel of nothing else is
    zero); the largest finite fp32 number stands for an infinite max|x|. ``paged_append`` keeps them page by page; this rebuilds
    them for pages that came from elsewhere (a copied prefix, a swapped-in sequence). A page that several
    sequences share is summarised once for each of them, so it should be full in all. Every column of the
    table is visited: pass it cut to the longest sequence where that is known.
    """
    rc = N.glue().paged_block_summary(k_cache, block_table,
                                      context_lens, k_scale, summary, summary_scale)
    if rc:
        N.check(rc, "bd_paged_block_summary")


def _check_row(q):
    if q.dim() not in (3, 4) or (q.dim() == 4 and q.shape[2] != 1):
        raise ValueError("q must be [B, H_q, D] or [B, H_q, 1, D]")


def paged_select_blocks(q, summary, summary_scale, block_table, context_lens, budget, block_size, *, sink_blocks=0,
                        recent_blocks=1):
    """Logical pages for one new token of each sequence, int32 [B, H_k, budget], ascending, -1 after the last.

    The ``sink_blocks`` first and ``recent_blocks`` last pages, then those with the largest estimate of q.k's
    maximum over the page (8-bit q and summaries, rounded to the nearest; the largest over the KV head's query
    heads, the lower page on ties). A q that is NaN counts as zero, an infinite one as the largest finite fp32
    number.
    """
    _check_row(q)
    if budget < 1:
        raise ValueError("budget must be at least one page")
    rc, selected = N.glue().paged_select(q, summary, summary_scale, block_table,
                                         context_lens, block_size, budget, sink_blocks,
                                         recent_blocks)
    if rc:
        N.check(rc, "bd_paged_select")
    return selected


def paged_decode_attn(q, k_cache, v_cache, block_table, context_lens, scaling, *, k_scale=1.0, v_scale=1.0,
                      selected=None, return_lse=False):
    """softmax(scaling * q.k) . v of one new token a sequence over its cached tokens.

    q [B, H_q, D] or [B, H_q, 1, D] (bf16 / f16 / f32) -> the same shape and type; query head h reads KV
    head h // (H_q / H_k). ``selected`` int32 [B, H_k, n] (as ``paged_select_blocks`` gives it) limits each KV
    head to those logical pages. Sequences without a token give zeros, and so do rows all of whose scores
    are -inf; a score that is NaN or +inf makes its row NaN. With ``return_lse`` also the natural log of the
    softmax denominator, f32 [B, H_q] (-inf for such rows of zeros), to join parts of a sequence held
    elsewhere.
    """
    _check_row(q)
    rc, out, lse = N.glue().paged_decode_attn(q, k_cache, v_cache, block_table,
                                              context_lens, selected, scaling, k_scale,
                                              v_scale, return_lse)
    if rc:
        N.check(rc, "bd_paged_decode_attn")
    return (out, lse) if return_lse else out


def paged_sparse_decode_attn(q, k_cache, v_cache, summary, summary_scale, block_table, context_lens, budget_blocks,
                             scaling, *, sink_blocks=0, recent_blocks=1, k_scale=1.0, v_scale=1.0,
                             return_selected=False):
    """``paged_decode_attn`` over the ``budget_blocks`` pages that ``paged_select_blocks`` chooses for each
    KV head; with ``return_selected`` (out, selected)."""
    _check_row(q)
    if budget_blocks < 1:
        raise ValueError("budget_blocks must be at least one page")
    rc, out, selected = N.glue().paged_sparse_decode_attn(
        q, k_cache, v_cache, summary, summary_scale, block_table,
        context_lens, budget_blocks, sink_blocks, recent_blocks, scaling, k_scale, v_scale)
    if rc:
        N.check(rc, "bd_paged_sparse_decode_attn")
    return (out, selected) if return_selected else out
