"""Attention weight of cached keys, and rows shortened to those that carry the most of it (no reference
counterpart: the reference's operator reads a cache that its caller keeps).

A decoder that bounds its cache keeps, for each layer, FP32 sums scores [rows, Hkv, S] (S at least
W * page_size): how much attention weight every cached key got, entry j of a row for its cache position
j. add_weights adds that of a step's new tokens; evict_rows drops the keys with the least of it.
"""
from __future__ import annotations

import math

import torch

from fgw_amd import _lib
from fgw_amd.operators.mha.kernels.mha_paged_decode_hip import _device_info

_kv = _lib.load_kv_module()


def add_weights(scores, q, k_cache, block_table, cache_seqlens, cu_seqlens, page_size, last, *, decay=1.0,
                softmax_scale=None):
    """Add the attention weight that cached keys get from new tokens to scores, in place.

    q, the pool, table and metadata are those of build_extend_kernel's callable (causal, no window), the
    new tokens' keys written already. For request b with n new tokens, K/V head h and key j < len,

      scores[b, h, j] = (decay * scores[b, h, j] if j < len - n else 0) + sum of softmax(scale q k^T)_j

    over the query heads of h and the last `last` of the new tokens (all, where they are fewer): 1 in a
    decode step, the prompt's length for all of a prompt, some tens for what its end looks back at. (No more
    than the longest request of the call has: the sizes of T and last say which kernels run, and a decode step
    with a last of some tens takes those of many rows, 2 to 2.5 times as long.) The
    keys of new tokens thus begin at zero without being cleared; decay 0 forgets all that was there.
    Requests without new tokens, and entries from len on, are left. Lengths and page ids out of range are
    taken as there; rows that see no key add nothing; a NaN in a query or in a key that it sees, or a score of plus
    infinity, gives NaN to all keys that it sees, and a key with a score of minus infinity gets nothing (a row with no
    other scores adds nothing). Sums are fp32, in the same order on every run. Nothing is read back: the call
    can be captured into a HIP graph. Records no gradient, and scores may require none.
    """
    if last < 1:
        raise ValueError("the number of tokens that count must be positive")
    if not (decay >= 0 and math.isfinite(decay)):
        raise ValueError("the decay must be finite and not negative")
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("the scale of the scores must be positive and finite")
    if q.device.type != "cuda":
        raise ValueError("contiguous inputs on the same GPU required")
    _kv.weights(scores, q, k_cache, block_table, cache_seqlens, cu_seqlens, page_size, min(last, 2**31 - 1), scale,
                decay, _device_info(q.device.index).num_cus)


def evict_rows(k_pools, v_pools, scores, refs, table, lens, keep, page_size, *, first=0, recent=0):
    """Shorten rows to the keys that carry the most attention weight, in every layer's pools.

    k_pools and v_pools [pages * page_size, Hkv, ...] and scores [rows, Hkv, S] are lists with an entry for
    each layer, refs, table and lens the books of cache_pages, keep int32 [rows]. Row r with lens[r] >
    keep[r] >= 0 keeps keep[r] tokens (others stay as they are): the first `first`, the last `recent` and,
    of those between, the ones with the largest scores, equal ones from the lowest position on and NaN as
    minus infinity. Each layer and K/V head chooses for itself; the kept tokens stay in order and move, with
    their scores, to the positions 0 .. keep[r] - 1, and lens[r] = keep[r]. Scores from there on are left,
    and so are the keys' rotary positions: later tokens take theirs from the caller (mha_paged_append's
    positions), no longer from the cache length.

    The tokens move to fresh pages, lowest id first and rows in order, from the page that holds token
    `first` on; whole pages before that stay, shared or not, and the pages that a row leaves lose a holder.
    Returns int32 [2]: rows refused for want of pages (that call for more, with the rows before them, than
    are free: what this call gives back is free for the next one), rows refused because keep is less than
    first + recent. Tokens of page ids outside the pools move as zeros. Every decision is made on the GPU, the
    same on every run; nothing is read back.
    """
    return _kv.evict(k_pools, v_pools, scores, refs, table, lens, keep, page_size, first, recent)
