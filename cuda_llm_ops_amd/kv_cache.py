"""The paged KV cache's operators, over the C ABI of include/fgqa_kv.h.

A paged cache is a pair of tensors [num_pages, page_size, Hkv, 128] (bf16,
torch.float8_e4m3fn or torch.int8) and a block table int32 [B, max_pages]: token
t of sequence b is slot t % page_size of page block_table[b, t // page_size].
8-bit caches hold codes; ``k_scale`` and ``v_scale`` are fp32 tensors
[num_pages, Hkv], a scale for each page of each KV head, or (float8_e4m3fn
only) two numbers for the whole cache.  A tensor of one element counts as a number
(the host reads it), unless both are the [num_pages, Hkv] scales of a cache of one
page and head.  Calls that write a cache (append, evict) refuse K and V caches or
scales that share memory.

    append_kv_paged              writes new tokens
    flash_gqa.decode_flash_gqa_paged   single-token attention
    accumulate_kv_weights_paged  the attention weight each cached token got
    evict_kv_paged               cuts sequences to a budget of tokens by weight

No counterpart in the reference.  PyTorch only provides device memory and the
current stream.  Every tensor of a call lives on one device; the call runs on that
device's current stream.
"""
from __future__ import annotations

import torch

from . import _lib
from .flash_gqa import PreparedLaunch, _get_device, _stream

__all__ = ["append_kv_paged", "accumulate_kv_weights_paged", "evict_kv_paged"]


class DeviceLaunch(PreparedLaunch):
    """A ``PreparedLaunch`` of an argument block's bytes, on the current stream of
    its tensors' device."""

    def __init__(self, fn, packed, keep, out, where, device):
        self._fn, self._args, self._keep, self._where = fn, packed, keep, where
        self._device = device
        self.out = out

    def __call__(self):
        if _get_device is None or self._device == _get_device():
            st = self._fn(self._args, _stream())
        else:
            with torch.cuda.device(self._device):
                st = self._fn(self._args, _stream())
        if st != _lib.FGQA_OK:
            raise _lib.FgqaError(st, self._where)
        return self.out


def call_native(name, device_of, *args):
    """A function of the native module (csrc/python/kv_native.cpp: the argument
    checks and the C ABI call), with the device of the tensor `device_of` current."""
    r = getattr(_lib.native(), name)(*args)
    if r is NotImplemented:   # another device than the current one
        with torch.cuda.device(device_of.device):
            r = getattr(_lib.native(), name)(*args)
    return r


def append_kv_paged(k, v, k_cache, v_cache, block_table, seqlens, new_lens=None, k_scale=1.0, v_scale=1.0):
    """Writes new tokens to a paged cache, in place; returns (k_cache, v_cache).

    k, v: bf16 [B, N, Hkv, 128], the new tokens; seqlens: int32 [B], tokens the
    sequences hold already (not changed); new_lens: int32 [B], how many of the N
    new ones are written (None: all).  Token i of row b becomes token
    seqlens[b] + i.  Tokens past the block table, and those of pages outside the
    cache, are not written; a page must not be written by two sequences of a call.

    With block scales, a block that gets its first slot gets the smallest power of
    two that brings its new tokens inside the codes' range (448 or 127); one that
    holds older tokens keeps its scale or grows it, and its older codes are rounded
    to the larger one.  Infinities become the largest code; NaN stays NaN in
    float8_e4m3fn and becomes 0 in int8.  With one scale for the cache, values are
    divided by it and saturated."""
    call_native("append", k, k, v, k_cache, v_cache, block_table, seqlens, new_lens, k_scale, v_scale)
    return k_cache, v_cache


def accumulate_kv_weights_paged(q, k_cache, lse, block_table, seqlens, weights, scale=None, k_scale=1.0,
                                max_seqlen=None):
    """Adds what one single-token attention gave each cached token to its weight,
    in place; returns ``weights``.

    weights[b, h, t] += sum over KV head h's query heads g of
    exp(scale * q[b, g] . K[b, t, h] - lse[b, g]) for t < seqlens[b].

    q: bf16 [B, Hq, 128]; lse: fp32 [B, Hq], as ``decode_flash_gqa_paged`` writes it
    for this q; weights: fp32 [B, Hkv, W], W >= max_seqlen (by default the block
    table's tokens or W, whichever is less: tokens from W on have no weight)."""
    call_native("weights", q, q, k_cache, lse, block_table, seqlens, weights, scale, k_scale, max_seqlen)
    return weights


def evict_kv_paged(k_cache, v_cache, block_table, seqlens, weights, new_block_table, budget, recent=0, k_scale=1.0,
                   v_scale=1.0, new_seqlens=None, new_weights=None, kept=None, max_seqlen=None):
    """Cuts each sequence to at most ``budget`` tokens, chosen for each KV head by
    its weights, and moves them to new pages; returns (new_seqlens, new_weights, kept).

    A longer sequence keeps its last ``recent`` tokens (at most budget) and, of
    those before, the ones of largest weight (of equal ones the lowest index; NaN
    counts as larger than any number), in order; a sequence of up to ``budget`` tokens keeps all.  Token
    kept[b, h, i] becomes token i, in page new_block_table[b, i // page_size].

    weights: fp32 [B, Hkv, W]; tokens from W on have none and are kept as the recent
    ones are.  With a ``max_seqlen`` (at most W), lengths are clamped to it.
    new_block_table: int32 [B, pages] for min(budget, W or max_seqlen) tokens; longer
    sequences are cut to what it holds.  new_seqlens: int32 [B]; new_weights: fp32
    [B, Hkv, W], the kept tokens' weights, then zeros; kept: int32
    [B, Hkv, budget], -1 past the kept tokens (each allocated when None).

    The new pages must be apart from every page that the call reads, and from each
    other.  The old pages stay as they are: free those that no other sequence
    shares.  Blocks with scales are scaled anew, as in ``append_kv_paged``."""
    return call_native("evict", k_cache, k_cache, v_cache, block_table, seqlens, weights, new_block_table, budget, recent,
                       k_scale, v_scale, new_seqlens, new_weights, kept, max_seqlen)
