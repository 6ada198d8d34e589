"""The paged KV cache's operators, over the C ABI of include/fgqa_kv.h.

A paged cache is a pair of tensors [num_pages, page_size, Hkv, 128] (bf16,
torch.float8_e4m3fn or torch.int8) and a block table int32 [B, max_pages]: token
t of sequence b is slot t % page_size of page block_table[b, t // page_size].
8-bit caches hold codes; ``k_scale`` and ``v_scale`` are fp32 tensors
[num_pages, Hkv], a scale for each page of each KV head, or (float8_e4m3fn
only) two numbers for the whole cache.

    append_kv_paged              writes new tokens
    flash_gqa.decode_flash_gqa_paged   single-token attention
    accumulate_kv_weights_paged  the attention weight each cached token got
    evict_kv_paged               cuts sequences to a budget of tokens by weight

No counterpart in the reference.  PyTorch only provides device memory and the
current stream.  Every tensor of a call lives on one device; the call runs on that
device's current stream.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .flash_gqa import PreparedLaunch, _get_device, _prep, _ptr, _require_cuda, _stream

__all__ = ["append_kv_paged", "accumulate_kv_weights_paged", "evict_kv_paged"]

_DTYPES = {torch.bfloat16: _lib.FGQA_KV_BF16, torch.float8_e4m3fn: _lib.FGQA_KV_FP8_E4M3,
           torch.int8: _lib.FGQA_KV_INT8}


class DeviceLaunch(PreparedLaunch):
    """A ``PreparedLaunch`` on the current stream of its tensors' device."""

    def __init__(self, fn, args, keep, out, where, device):
        super().__init__(fn, args, keep, out, where)
        self._device = device.index

    def __call__(self):
        _launch(self._fn, self._ref, self._device, self._where)
        return self.out


def _launch(fn, ref, device, where):
    if _get_device is None or device == _get_device():
        st = fn(ref, _stream())
    else:
        with torch.cuda.device(device):
            st = fn(ref, _stream())
    if st != _lib.FGQA_OK:
        raise _lib.FgqaError(st, where)


# --------------------------------------------------------------------------- checks
def _rows_apart(t) -> bool:
    """No two elements of t share memory (an expanded tensor's do)."""
    if t.is_contiguous():
        return True
    end = 1   # elements that the dims so far span
    for st, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if st < end:
            return False
        end += st * (n - 1)
    return True


def _meet(a, b) -> bool:
    """The address ranges of a and b overlap."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (
            1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0)
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def check_device(first, *others) -> None:
    """All tensors on the GPU of the first."""
    _require_cuda(first)
    for t in others:
        if isinstance(t, torch.Tensor) and t.device != first.device:
            raise ValueError(f"all tensors must be on {first.device}, got one on {t.device}")


def check_table(table, B, name) -> int:
    """Row stride of a block table."""
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B \
            or (table.shape[1] > 1 and B > 0 and table.stride(1) != 1):
        raise ValueError(f"{name} must be an int32 [B, max_pages] tensor with contiguous rows")
    return table.stride(0) if B > 1 else table.shape[1]


def check_lens(lens, B, name) -> None:
    if lens.dtype != torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [B] tensor")


def check_max_seqlen(max_seqlen, table, page_size) -> int:
    most = table.shape[1] * page_size
    if max_seqlen is None:
        return most
    if not 0 <= int(max_seqlen) <= most:
        raise ValueError("max_seqlen must be between 0 and the block table's tokens")
    return int(max_seqlen)


def _check_cache(cache, name):
    if cache.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bf16, float8_e4m3fn or int8")
    if cache.dim() != 4:
        raise ValueError(f"{name} must be [num_pages, page_size, Hkv, D]")
    num_pages, page_size, Hkv, D = cache.shape
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two")
    if D != 128 or Hkv < 1:
        raise ValueError("head_dim must be 128 on this path")
    if cache.stride(3) != 1:
        raise ValueError("the caches' head_dim must be contiguous")
    per_16 = 16 // cache.element_size()
    if cache.data_ptr() & 15 or any(s % per_16 for s in cache.stride()[:3]):
        raise ValueError(f"{name} must be 16-byte aligned, with strides in multiples of 16 bytes")


def _scale_fields(cache, scale, name):
    """(address, number, strides) of a scale: block scales or one for the cache."""
    if isinstance(scale, torch.Tensor):
        if cache.dtype == torch.bfloat16:
            raise ValueError("bf16 caches have no block scales")
        if scale.dtype != torch.float32 or scale.shape != (cache.shape[0], cache.shape[2]):
            raise ValueError(f"{name} must be an fp32 [num_pages, Hkv] tensor")
        return scale.data_ptr(), 1.0, scale.stride()
    if cache.dtype == torch.int8:
        raise ValueError(f"int8 caches need {name} as an fp32 [num_pages, Hkv] tensor")
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{name} must be finite")
    if cache.dtype == torch.bfloat16 and scale != 1.0:
        raise ValueError("bf16 caches have no scale")
    return 0, scale, (0, 0)


def cache_fields(k_cache, v_cache, k_scale, v_scale):
    """The values of ``_lib._KV_CACHE``; v_cache None: a call that reads K only."""
    _check_cache(k_cache, "k_cache")
    ks = _scale_fields(k_cache, k_scale, "k_scale")
    if v_cache is None:
        vs, vp, vst = (0, 1.0, (0, 0)), 0, (0, 0, 0)
    else:
        if v_cache.dtype != k_cache.dtype or v_cache.shape != k_cache.shape:
            raise ValueError("k_cache and v_cache must share dtype and shape")
        _check_cache(v_cache, "v_cache")
        vs, vp, vst = _scale_fields(v_cache, v_scale, "v_scale"), v_cache.data_ptr(), v_cache.stride()[:3]
        if isinstance(k_scale, torch.Tensor) != isinstance(v_scale, torch.Tensor):
            raise ValueError("k_scale and v_scale must both be tensors or both numbers")
    num_pages, page_size, Hkv, D = k_cache.shape
    return (k_cache.data_ptr(), vp, ks[0], vs[0], _DTYPES[k_cache.dtype], Hkv, D, page_size, num_pages, ks[1], vs[1],
            *k_cache.stride()[:3], *vst, *ks[2], *vs[2])


def _check_written(*ts):
    for t in ts:
        if isinstance(t, torch.Tensor) and not _rows_apart(t):
            raise ValueError("a tensor that is written must not overlap itself (expanded dims)")


# --------------------------------------------------------------------------- append
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
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("append expects bf16 tokens")
    cache = cache_fields(k_cache, v_cache, k_scale, v_scale)
    if k.dim() != 4 or k.shape != v.shape or k.shape[2:] != k_cache.shape[2:]:
        raise ValueError("K and V must be [B, N, Hkv, D] matching the caches")
    if not isinstance(k_scale, torch.Tensor) and not (k_scale > 0 and v_scale > 0):
        raise ValueError("k_scale and v_scale must be positive")
    B, N = k.shape[:2]
    table_stride = check_table(block_table, B, "block_table")
    check_lens(seqlens, B, "seqlens")
    if new_lens is not None:
        check_lens(new_lens, B, "new_lens")
    _check_written(k_cache, v_cache, k_scale, v_scale)
    check_device(k, v, k_cache, v_cache, block_table, seqlens, new_lens, k_scale, v_scale)
    k, v = _prep(k), _prep(v)
    a = _lib.pack_kv_append(*cache, _ptr(k), _ptr(v), *k.stride()[:3], *v.stride()[:3], _ptr(block_table),
                            table_stride, _ptr(seqlens), _ptr(new_lens), B, N, block_table.shape[1])
    _launch(_lib.lib().fgqa_kv_append, ctypes.byref(a), k.device.index, "fgqa_kv_append")
    return k_cache, v_cache


# --------------------------------------------------------------------------- weights
def accumulate_kv_weights_paged(q, k_cache, lse, block_table, seqlens, weights, scale=None, k_scale=1.0,
                                max_seqlen=None):
    """Adds what one single-token attention gave each cached token to its weight,
    in place; returns ``weights``.

    weights[b, h, t] += sum over KV head h's query heads g of
    exp(scale * q[b, g] . K[b, t, h] - lse[b, g]) for t < seqlens[b].

    q: bf16 [B, Hq, 128]; lse: fp32 [B, Hq], as ``decode_flash_gqa_paged`` writes it
    for this q; weights: fp32 [B, Hkv, W], W >= max_seqlen (by default the block
    table's tokens or W, whichever is less)."""
    if q.dtype != torch.bfloat16 or q.dim() != 3:
        raise ValueError("expected a bf16 query [B, Hq, D]")
    cache = cache_fields(k_cache, None, k_scale, None)
    B, Hq, D = q.shape
    _, page_size, Hkv, _ = k_cache.shape
    if k_cache.shape[3] != D:
        raise ValueError("the cache's head_dim must match Q")
    if Hq < 1 or Hq % Hkv != 0:
        raise ValueError("Query heads must be divisible by KV heads")
    if lse.dtype != torch.float32 or lse.shape != (B, Hq) or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 [B, Hq] tensor")
    _check_weights(weights, B, Hkv, "weights")
    table_stride = check_table(block_table, B, "block_table")
    check_lens(seqlens, B, "seqlens")
    if max_seqlen is None:
        max_seqlen = min(block_table.shape[1] * page_size, weights.shape[2])
    max_seqlen = check_max_seqlen(max_seqlen, block_table, page_size)
    if weights.shape[2] < max_seqlen:
        raise ValueError("weights must hold max_seqlen tokens")
    _check_written(weights)
    check_device(q, k_cache, lse, block_table, seqlens, weights, k_scale)
    q = _prep(q)
    a = _lib.pack_kv_weights(*cache, _ptr(q), _ptr(lse), _ptr(weights), *q.stride()[:2], *weights.stride()[:2],
                             _ptr(block_table), table_stride, _ptr(seqlens), B, max_seqlen, Hq,
                             1.0 / math.sqrt(D) if scale is None else float(scale))
    _launch(_lib.lib().fgqa_kv_weights, ctypes.byref(a), q.device.index, "fgqa_kv_weights")
    return weights


def _check_weights(w, B, Hkv, name):
    if w.dtype != torch.float32 or w.dim() != 3 or w.shape[:2] != (B, Hkv) or (w.numel() > 1 and w.shape[2] > 1 and w.stride(2) != 1):
        raise ValueError(f"{name} must be an fp32 [B, Hkv, W] tensor with contiguous rows")


# --------------------------------------------------------------------------- evict
def evict_kv_paged(k_cache, v_cache, block_table, seqlens, weights, new_block_table, budget, recent=0, k_scale=1.0,
                   v_scale=1.0, new_seqlens=None, new_weights=None, kept=None, max_seqlen=None):
    """Cuts each sequence to at most ``budget`` tokens, chosen for each KV head by
    its weights, and moves them to new pages; returns (new_seqlens, new_weights, kept).

    A longer sequence keeps its last ``recent`` tokens (at most budget) and, of
    those before, the ones of largest weight (of equal ones the lowest index; NaN
    counts as larger than any number), in order; a sequence of up to ``budget`` tokens keeps all.  Token
    kept[b, h, i] becomes token i, in page new_block_table[b, i // page_size].

    weights: fp32 [B, Hkv, W], W >= max_seqlen (by default the block table's tokens
    or W, whichever is less); new_block_table: int32 [B, pages] for
    min(budget, max_seqlen) tokens.  new_seqlens: int32 [B]; new_weights: fp32
    [B, Hkv, W], the kept tokens' weights, then zeros; kept: int32
    [B, Hkv, budget], -1 past the kept tokens (each allocated when None).

    The new pages must be apart from every page that the call reads, and from each
    other.  The old pages stay as they are: free those that no other sequence
    shares.  Blocks with scales are scaled anew, as in ``append_kv_paged``."""
    cache = cache_fields(k_cache, v_cache, k_scale, v_scale)
    _, page_size, Hkv, _ = k_cache.shape
    budget, recent = int(budget), int(recent)
    if budget < 1 or recent < 0:
        raise ValueError("budget must be positive and recent not negative")
    if seqlens.dim() != 1:
        raise ValueError("seqlens must be a contiguous int32 [B] tensor")
    B = seqlens.shape[0]
    check_lens(seqlens, B, "seqlens")
    _check_weights(weights, B, Hkv, "weights")
    W = weights.shape[2]
    table_stride = check_table(block_table, B, "block_table")
    new_stride = check_table(new_block_table, B, "new_block_table")
    if max_seqlen is None:
        max_seqlen = min(block_table.shape[1] * page_size, W)
    max_seqlen = check_max_seqlen(max_seqlen, block_table, page_size)
    if W < max_seqlen:
        raise ValueError("weights must hold max_seqlen tokens")
    if new_block_table.shape[1] * page_size < min(budget, max_seqlen):
        raise ValueError("new_block_table must have pages for min(budget, max_seqlen) tokens")
    if new_seqlens is not None:
        check_lens(new_seqlens, B, "new_seqlens")
    if new_weights is not None:
        _check_weights(new_weights, B, Hkv, "new_weights")
        if new_weights.shape[2] != W:
            raise ValueError("new_weights must have weights' shape")
    if kept is not None and (kept.dtype != torch.int32 or kept.shape != (B, Hkv, budget) or not kept.is_contiguous()):
        raise ValueError("kept must be a contiguous int32 [B, Hkv, budget] tensor")
    _check_written(k_cache, v_cache, k_scale, v_scale, new_weights)
    given = [t for t in (new_seqlens, new_weights, kept) if t is not None]
    if any(_meet(t, x) for i, t in enumerate(given)
           for x in (*given[:i], weights, seqlens, block_table, new_block_table)):
        raise ValueError("new_seqlens, new_weights and kept must be apart from each other and from the inputs")
    check_device(k_cache, v_cache, block_table, seqlens, weights, new_block_table, k_scale, v_scale, new_seqlens,
                 new_weights, kept)
    dev = k_cache.device
    if new_seqlens is None:
        new_seqlens = torch.empty((B,), device=dev, dtype=torch.int32)
    if new_weights is None:
        new_weights = torch.empty((B, Hkv, W), device=dev, dtype=torch.float32)
    if kept is None:
        kept = torch.empty((B, Hkv, budget), device=dev, dtype=torch.int32)
    a = _lib.pack_kv_evict(*cache, _ptr(weights), _ptr(new_weights), *weights.stride()[:2], *new_weights.stride()[:2],
                           _ptr(block_table), _ptr(new_block_table), table_stride, new_stride, _ptr(seqlens),
                           _ptr(new_seqlens), _ptr(kept), B, max_seqlen, W, budget, recent)
    _launch(_lib.lib().fgqa_kv_evict, ctypes.byref(a), dev.index, "fgqa_kv_evict")
    return new_seqlens, new_weights, kept
