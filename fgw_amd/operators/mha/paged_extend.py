"""New tokens over the paged cache: their cache write and their attention, with grouped heads and
ragged counts (no reference counterpart: the reference's operator reads a cache that its caller
has written, with one K/V head per query head and the same number of queries in every request).

The new tokens of all requests are packed: request b has rows cu_seqlens[b] .. cu_seqlens[b + 1] of
Q [T, Hq, D] and K, V [T, Hkv, D] (int32 [B + 1], from 0, never falling), and its cache length
(cache_seqlens [B], int32) counts them, so its row j has the cache position len - n + j. The pool
K, V [N, Hkv, D], the block table [B, W] and the page size are those of mha_paged_decode. Rows at
and behind cu_seqlens[B] (a padded batch) are neither read nor written. A serving step is

  cache_pages.reserve_rows(...)           pages for the new tokens
  q = mha_paged_append(q, k, v, ...)      Q rotated, K rotated and V written to their pages
  o = kernel(q, k_cache, v_cache, ...)    build_extend_kernel's callable

with nothing read back from the device: every call can be captured into a HIP graph and replayed
after lengths, counts and tables were changed in place. Inference only: no gradient is recorded, and
none of the pools and outputs that a call writes may require one (torch.no_grad() lifts that).
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

from fgw_amd import _lib
from fgw_amd.operators.mha.kernels.mha_paged_decode_hip import _device_info, _dtype_name
from fgw_amd.operators.mha.rotary import Rotary

_kv = _lib.load_kv_module()


def mha_paged_append(q, k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, page_size, *,
                     rotary=None, positions=None, q_out=None):
    """Write the new tokens' K and V to their pages and return Q, both Q and K rotated.

    q [T, Hq, D], k and v [T, Hkv, D]: FP16 or BF16 rows, strides multiples of 16 bytes (views of
    one fused projection will do). Row cu_seqlens[b] + j goes to the pool row
    block_table[b, pos // page_size] * page_size + pos % page_size of its cache position pos; it is
    not written where pos lies outside [0, W * page_size) or the page id outside the pool (lengths are
    taken as given here; the attention clamps them). rotary (a Rotary) turns q and k to their cache
    positions, or to positions [T] (int32 or int64); None writes k as it is and copies q. Returns
    q_out ([T, Hq, D]; q itself for in place) or a new contiguous tensor. No two tokens may have the
    same cache position of one page. The two pools and q_out share no memory with each other or with
    anything the call reads (but q_out with q, as q itself); heads side by side in one buffer do not.
    """
    if rotary is None:
        if positions is not None:
            raise ValueError("positions need a rotary")
        return _kv.append(q, k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, page_size,
                          None, 0, 0, 1.0, None, q_out)
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    return _kv.append(q, k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, page_size,
                      rotary.turns, rotary.dim, rotary.interleaved, rotary.scale, positions, q_out)


class _ExtendKernel:
    """Launch callable of build_extend_kernel."""

    def __init__(self, heads, kv_heads, dim, page_size, dtype_name, device_index, is_causal, window,
                 softmax_scale):
        self.heads, self.kv_heads, self.dim, self.page_size = heads, kv_heads, dim, page_size
        self.dtype = torch.bfloat16 if dtype_name == "bfloat16" else torch.float16
        self.is_causal, self.window, self.softmax_scale = is_causal, window, softmax_scale
        self._tail = (page_size, heads, kv_heads, dim, dtype_name == "bfloat16", device_index, is_causal,
                      window or 0, softmax_scale, _device_info(device_index).num_cus)

    def __call__(self, q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, max_new, out=None):
        """O [T, Hq, D] (a new tensor, or `out`, contiguous and apart from all inputs). max_new: at
        least the new tokens of every request; the rows of a request's tokens past it are left as
        they are."""
        return _kv.extend(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, max_new,
                          *self._tail, out)


@lru_cache(maxsize=128)
def _planned(heads, kv_heads, dim, page_size, name, device_index, is_causal, window, scale):
    return _ExtendKernel(heads, kv_heads, dim, page_size, name, device_index, is_causal, window, scale)


def build_extend_kernel(heads, kv_heads, dim, page_size, dtype, device_index=None, *, is_causal=True,
                        window=None, softmax_scale=None):
    """Launch callable of the attention of new tokens over the paged cache.

    heads query heads over kv_heads K/V heads (query head h reads K/V head h // (heads //
    kv_heads)), D 16..256 in steps of 16, FP16 or BF16. is_causal: the token at cache position p
    sees the keys 0 .. p, with window (>= 1) only the last `window` of them, itself among them; not
    causal: every live key (attention over an encoder's cached states). softmax_scale: D ** -0.5
    unless given. The callable takes (q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens,
    max_new, out=None), shapes free from call to call, and reads nothing back. Lengths outside
    [0, W * page_size] are clamped (positions then follow from the clamped length, other ones than
    mha_paged_append wrote); tokens that see no key give zero rows; page ids outside the pool read as
    zeros. Keys that no token of a request sees do not matter, whatever they hold. A NaN in a query or
    in a key that it sees gives a row of NaN. A key whose V is not finite gives NaN or infinities to
    the tokens that see it, and may give NaN to other new tokens of the same request and call (a
    weight of 0 times it).
    """
    name = _dtype_name(dtype)
    if dim < 16 or dim > 256 or dim % 16:
        raise ValueError("D must be in [16, 256] and divisible by 16")
    if page_size <= 0:
        raise ValueError("positive page size, whole pool pages and positive table width required")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise ValueError("query heads must be a positive multiple of the K/V heads")
    if window is not None and (window < 1 or not is_causal):
        raise ValueError("a window must be positive and needs causal attention")
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("the scale of the scores must be positive and finite")
    if device_index is None:
        device_index = torch.cuda.current_device()
    return _planned(int(heads), int(kv_heads), int(dim), int(page_size), name, int(device_index),
                    bool(is_causal), None if window is None else min(int(window), 2**31 - 1), scale)


def mha_paged_extend(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, page_size,
                     is_causal=True, *, window=None, softmax_scale=None, out=None):
    """Attention of new tokens over the paged cache in one call, with its metadata checked.

    As build_extend_kernel's callable, after one copy of lengths and offsets to the host:
    0 <= len <= W * page_size, offsets from 0 to at most T and never falling.
    """
    if q.ndim != 3 or k_cache.ndim != 3:
        raise ValueError("expected Q[T,Hq,D], K/V[N,Hkv,D]")
    if block_table.ndim != 2 or cache_seqlens.ndim != 1 or cu_seqlens.ndim != 1:
        raise ValueError("metadata shape mismatch")
    if cache_seqlens.shape[0] != block_table.shape[0] or cu_seqlens.shape[0] != block_table.shape[0] + 1:
        raise ValueError("metadata shape mismatch")
    if block_table.dtype != torch.int32 or cache_seqlens.dtype != torch.int32 or cu_seqlens.dtype != torch.int32:
        raise ValueError("int32 metadata required")
    if q.device.type != "cuda" or any(x.device != q.device for x in (
            k_cache, v_cache, block_table, cache_seqlens, cu_seqlens)):
        raise ValueError("contiguous inputs on the same GPU required")
    kernel = build_extend_kernel(q.shape[1], k_cache.shape[1], q.shape[2], page_size, q.dtype,
                                 q.device.index, is_causal=is_causal, window=window,
                                 softmax_scale=softmax_scale)
    host = torch.cat((cache_seqlens, cu_seqlens)).tolist()
    batch = block_table.shape[0]
    lengths, cu = host[:batch], host[batch:]
    if batch == 0 or min(lengths) < 0 or max(lengths) > block_table.shape[1] * page_size:
        raise ValueError("Cache lengths must be within table capacity")
    news = [b - a for a, b in zip(cu, cu[1:])]
    if cu[0] != 0 or min(news) < 0 or cu[-1] > q.shape[0]:
        raise ValueError("cu_seqlens must run from 0 to at most T and never fall")
    return kernel(q, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens, max(1, max(news)), out)
