"""Attention of new tokens over the paged cache where groups of requests share a long prefix: samples or
beams of one prompt (cache_pages.fork_rows), requests behind one system prompt (no reference
counterpart: the reference's operator reads every request's whole cache).

Requests, packing, pools and metadata are those of paged_extend. Beside them, int32 on the GPU:

  cu_groups   [G + 1]  group g is the requests cu_groups[g] .. cu_groups[g + 1] (from 0, never falling;
                       requests behind the last group share nothing)
  prefix_lens [G]      keys that the requests of a group have in common, from cache position 0

A group's prefix is read through the table row of its first request, once for all its tokens; the other
rows hold the same keys, in the same pages (as a fork leaves the whole pages) or in copies of them. It
counts as far as the first request has it before its own new tokens. A request whose new tokens begin
within the prefix, or that is alone in its group, reads its own keys instead: the result is that of
paged_extend for any lengths, up to the order of fp32 sums. The prefix's softmax weights are held in two numbers of
the input type, as those of few new tokens are there. Inference only, as there.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from fgw_amd import _lib
from fgw_amd.operators.mha.paged_extend import build_extend_kernel

_kv = _lib.load_kv_module()


class _SharedKernel:
    """Launch callable of build_shared_kernel."""

    def __init__(self, extend, always):
        self.always = always
        self.heads, self.kv_heads, self.dim, self.page_size = (extend.heads, extend.kv_heads, extend.dim,
                                                               extend.page_size)
        self.dtype, self.softmax_scale = extend.dtype, extend.softmax_scale
        self._tail = extend._tail

    def __call__(self, q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, cu_groups, prefix_lens,
                 max_new, out=None):
        """O [T, Hq, D] (a new tensor, or `out`, contiguous and apart from all inputs). max_new: as in
        build_extend_kernel's callable."""
        return _kv.shared(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, cu_groups, prefix_lens,
                          self.always, max_new, *self._tail, out)


@lru_cache(maxsize=128)
def _planned(extend, always):
    return _SharedKernel(extend, always)


def build_shared_kernel(heads, kv_heads, dim, page_size, dtype, device_index=None, *, softmax_scale=None,
                        always=False):
    """Launch callable of the causal attention of new tokens where requests share prefixes.

    Heads, head dims, types and scale are those of build_extend_kernel. Sharing takes a second pass: a call
    whose prefixes are too short for that, by their lengths on the device, or whose requests have too many
    new tokens each, reads every request's keys itself, unless always is set. The callable takes (q, k_cache,
    v_cache, block_table, cache_seqlens, cu_seqlens, cu_groups, prefix_lens, max_new, out=None), shapes
    free from call to call, and reads nothing back: it can be captured into a HIP graph and replayed after
    lengths, groups and tables were changed in place. What build_extend_kernel says of lengths out of
    range, page ids outside the pool, NaN and infinities holds here too, for the tokens of a group in the
    place of those of a request.
    """
    return _planned(build_extend_kernel(heads, kv_heads, dim, page_size, dtype, device_index,
                                        softmax_scale=softmax_scale), bool(always))


def mha_paged_shared(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, cu_groups, prefix_lens,
                     page_size, *, softmax_scale=None, always=False, out=None):
    """Attention of new tokens with shared prefixes in one call, with its metadata checked.

    As build_shared_kernel's callable, after one copy of lengths and offsets to the host:
    0 <= len <= W * page_size; offsets of tokens from 0 to at most T and of groups from 0 to at most B,
    never falling; 0 <= prefix_lens.
    """
    if q.ndim != 3 or k_cache.ndim != 3:
        raise ValueError("expected Q[T,Hq,D], K/V[N,Hkv,D]")
    meta = (cache_seqlens, cu_seqlens, cu_groups, prefix_lens)
    if block_table.ndim != 2 or any(x.ndim != 1 for x in meta):
        raise ValueError("metadata shape mismatch")
    batch, groups = block_table.shape[0], prefix_lens.shape[0]
    if cache_seqlens.shape[0] != batch or cu_seqlens.shape[0] != batch + 1 or cu_groups.shape[0] != groups + 1:
        raise ValueError("metadata shape mismatch")
    if any(x.dtype != torch.int32 for x in (block_table, *meta)):
        raise ValueError("int32 metadata required")
    if q.device.type != "cuda" or any(x.device != q.device for x in (k_cache, v_cache, block_table, *meta)):
        raise ValueError("contiguous inputs on the same GPU required")
    kernel = build_shared_kernel(q.shape[1], k_cache.shape[1], q.shape[2], page_size, q.dtype, q.device.index,
                                 softmax_scale=softmax_scale, always=always)
    host = torch.cat(meta).tolist()
    lengths, host = host[:batch], host[batch:]
    cu, host = host[:batch + 1], host[batch + 1:]
    first, prefixes = host[:groups + 1], host[groups + 1:]
    if batch == 0 or min(lengths) < 0 or max(lengths) > block_table.shape[1] * page_size:
        raise ValueError("Cache lengths must be within table capacity")
    news = [b - a for a, b in zip(cu, cu[1:])]
    if cu[0] != 0 or min(news) < 0 or cu[-1] > q.shape[0]:
        raise ValueError("cu_seqlens must run from 0 to at most T and never fall")
    if first[0] != 0 or any(a > b for a, b in zip(first, first[1:])) or first[-1] > batch:
        raise ValueError("cu_groups must run from 0 to at most B and never fall")
    if any(n < 0 for n in prefixes):
        raise ValueError("prefix lengths must not be negative")
    return kernel(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, cu_groups, prefix_lens,
                  max(1, max(news)), out)
