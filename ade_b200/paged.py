"""Paged key-value cache for batches of independent requests.

A cache layer is a pair of arrays (pages, kv_heads, page_size, head_dim); a request owns a list of pages, its row of a block table
that all layers share, so requests of any lengths live in one cache, enter and leave it at any time, and take memory by the
page.  Lengths, tables and the stack of free pages stay on the device: a step captured in a CUDA graph follows them.  The three
launches of a step:

    slots, positions, requests, ... = paged_extend(lengths, new_tokens, block_table, free_pages, free_count, rows, page_size)
    paged_write(k, v, slots, k_pages, v_pages, cos, sin)                                         # per layer
    out = paged_attn_decode(q, block_table, requests, positions, k_pages, v_pages, scale, cos, sin)

The reference has no counterpart: it generates with ``model.generate`` of transformers (src/evaluate.py:241), on one contiguous cache for
a batch of equal lengths, which ``decode_ops.attn_decode`` serves.
"""
from __future__ import annotations

import torch

from .kernels import _call

MAX_REQUESTS = 4096            # ADE_B200_MAX_REQUESTS


def paged_extend(lengths: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                 total: int, page_size: int, in_place: bool = False):
    """Make room for new tokens: pages from the stack of free ones, entries of the block table, and where each token goes.

    Parameters:
        lengths: (B,) int32, the tokens each request has; B <= 4096.
        new_tokens: (B,) int32, how many to add; 0: none; negative: the request ends, its pages go back before any is taken.
        block_table: (B, width) int32, written: new pages are entered behind those a request has.
        free_pages, free_count: (pages,) and (1,) int32, the stack of free pages (written) and its height.
        total: rows of the packed batch of new tokens, request after request; at least their number.
        page_size: tokens per page.
        in_place: write the new lengths and height into `lengths` and `free_count` instead of new tensors.

    Returns:
        (slots, positions, requests, lengths, free_count, status): for each of the `total` rows the slot (page * page_size + offset, int64),
        the position in its request (int64) and the request (int32); rows behind the last token, and those of a request that
        could not grow, have slot -1, position 0, request -1.  status (B,) int32 is 0, or a key of ``_lib.PAGED_STATUS`` that says
        why the request did not grow; its length then stays as it was.  Where `total` is too small, every request behind the first
        that did not fit has ADE_PAGED_NO_ROW, one without new tokens too.  The returned tensors share one allocation: whoever
        keeps, saves or resizes one of them by itself takes a clone.
    """
    out = _call("paged_extend", lengths, new_tokens, block_table, free_pages, free_count, total, page_size, in_place)
    return (*out[:3], lengths, free_count, out[5]) if in_place else out


def paged_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None) -> None:
    """Keys and values of new tokens into the pages of one layer.

    k and v are (rows, kv_heads, head_dim) bfloat16 views with a contiguous last dimension and any other strides; slots (rows,) int64 from
    `paged_extend`.  With cos and sin, (rows, head_dim), keys are rotated in float32 and rounded once (transformers rotates in bfloat16
    and rounds three times, so last bits differ from its cache); without, they are stored as they are.  Rows whose slot is no place of the cache are left out.  head_dim: a multiple of 32 up to 256.
    """
    _call("paged_write", k, v, slots, k_pages, v_pages, cos, sin)


def paged_attn_decode(q: torch.Tensor, block_table: torch.Tensor, requests: torch.Tensor, positions: torch.Tensor, k_pages: torch.Tensor,
                      v_pages: torch.Tensor, scale: float, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q K^T scale) V of single token rows over the cached positions 0 .. positions[t] of request requests[t].

    q is a (rows, q_heads, head_dim) bfloat16 view with a contiguous last dimension, rotated with cos and sin where they are given; the
    heads of a key-value head are consecutive.  Rows without a request (requests[t] = -1) are zero.  Positions whose table entry is no page
    are left out.  What a row sees of keys, values and scores has to be finite; where it is not, that row (and no other) may be NaN.  What
    stands behind positions[t] is not read.  Returns (rows, q_heads * head_dim) bfloat16; scores, probabilities and sums are float32.
    """
    return _call("paged_attn", q, block_table, requests, positions, k_pages, v_pages, scale, cos, sin)
