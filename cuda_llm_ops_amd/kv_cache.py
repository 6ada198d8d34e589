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

import math

import torch

from . import _lib
from .flash_gqa import PreparedLaunch, _get_device, _prep, _require_cuda, _stream

__all__ = ["append_kv_paged", "accumulate_kv_weights_paged", "evict_kv_paged"]

# C ABI type and, less one, the elements of 16 bytes
_DTYPES = {torch.bfloat16: (_lib.FGQA_KV_BF16, 7), torch.float8_e4m3fn: (_lib.FGQA_KV_FP8_E4M3, 15),
           torch.int8: (_lib.FGQA_KV_INT8, 15)}


class DeviceLaunch(PreparedLaunch):
    """A ``PreparedLaunch`` on the current stream of its tensors' device."""

    def __init__(self, fn, packed, keep, out, where, device):
        self._fn, self._args, self._keep, self._where = fn, packed, keep, where
        self._device = device
        self.out = out

    def __call__(self):
        launch(self._fn, self._args, self._device, self._where)
        return self.out


def launch(fn, packed, device, where):
    """Calls the C ABI with an argument block's bytes on the device's current stream."""
    if _get_device is None or device == _get_device():
        st = fn(packed, _stream())
    else:
        with torch.cuda.device(device):
            st = fn(packed, _stream())
    if st != 0:
        raise _lib.FgqaError(st, where)


# --------------------------------------------------------------------------- checks
# (A single-token step is a few microseconds of GPU work: the checks that pass
# read each property of a tensor once and name what is wrong only afterwards.)
def _rows_apart(t) -> bool:
    """No two elements of t share memory (an expanded tensor's do)."""
    end = 1   # elements that the dims so far span
    for st, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if st < end:
            return False
        end += st * (n - 1)
    return True


def _check_written(*ts):
    for t in ts:
        if not (t.is_contiguous() or _rows_apart(t)):
            raise ValueError("a tensor that is written must not overlap itself (expanded dims)")


def _meet(a, b) -> bool:
    """The address ranges of a and b overlap."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (
            1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0)
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def check_device(first, *others) -> int:
    """All tensors on one GPU; its index."""
    dev = first.get_device()
    if dev < 0:
        _require_cuda(first)
    for t in others:
        if t.get_device() != dev:
            raise ValueError(f"all tensors must be on {first.device}, got one on {t.device}")
    return dev


def check_table(table, B, name):
    """(pages of a row, stride of the rows) of a block table."""
    shape, st = table.shape, table.stride()
    if table.dtype is not torch.int32 or len(shape) != 2 or shape[0] != B or (st[1] != 1 and shape[1] > 1 and B > 0):
        raise ValueError(f"{name} must be an int32 [B, max_pages] tensor with contiguous rows")
    return shape[1], st[0] if B > 1 else shape[1]


def check_lens(lens, B, name) -> None:
    if lens.dtype is not torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [B] tensor")


def check_max_seqlen(max_seqlen, most) -> int:
    max_seqlen = int(max_seqlen)
    if not 0 <= max_seqlen <= most:
        raise ValueError("max_seqlen must be between 0 and the block table's tokens")
    return max_seqlen


def _refuse_cache(cache, name):
    if cache.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bf16, float8_e4m3fn or int8")
    if cache.dim() != 4:
        raise ValueError(f"{name} must be [num_pages, page_size, Hkv, D]")
    _, page_size, Hkv, D = cache.shape
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two")
    if D != 128 or Hkv < 1:
        raise ValueError("head_dim must be 128 on this path")
    if cache.stride(3) != 1:
        raise ValueError("the caches' head_dim must be contiguous")
    raise ValueError(f"{name} must be 16-byte aligned, with strides in multiples of 16 bytes")


def _cache_layout(cache, name):
    """(code, shape, address, strides) of a cache."""
    known, shape, st, p = _DTYPES.get(cache.dtype), cache.shape, cache.stride(), cache.data_ptr()
    if known is None or len(shape) != 4:
        _refuse_cache(cache, name)
    code, mask = known
    _, P, Hkv, D = shape
    if D != 128 or Hkv < 1 or P < 1 or P & (P - 1) or st[3] != 1 or p & 15 or (st[0] | st[1] | st[2]) & mask:
        _refuse_cache(cache, name)
    return code, shape, p, st


def _block_scales(scale, dtype, shape, name):
    """(address, strides) of a tensor of block scales."""
    if dtype is torch.bfloat16:
        raise ValueError("bf16 caches have no block scales")
    s = scale.shape
    if scale.dtype is not torch.float32 or len(s) != 2 or s[0] != shape[0] or s[1] != shape[2]:
        raise ValueError(f"{name} must be an fp32 [num_pages, Hkv] tensor")
    return scale.data_ptr(), scale.stride()


def _whole_scale(scale, dtype, name):
    if dtype is torch.int8:
        raise ValueError(f"int8 caches need {name} as an fp32 [num_pages, Hkv] tensor")
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{name} must be finite")
    if dtype is torch.bfloat16 and scale != 1.0:
        raise ValueError("bf16 caches have no scale")
    return scale


def cache_fields(k_cache, v_cache, k_scale, v_scale):
    """(the values of ``_lib._KV_CACHE``, whether there are block scales)."""
    code, shape, kp, kst = _cache_layout(k_cache, "k_cache")
    dtype = k_cache.dtype
    if v_cache.dtype is not dtype or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must share dtype and shape")
    _, _, vp, vst = _cache_layout(v_cache, "v_cache")
    blocks = isinstance(k_scale, torch.Tensor)
    if blocks != isinstance(v_scale, torch.Tensor):
        if dtype is torch.int8:
            _whole_scale(v_scale if blocks else k_scale, dtype, "v_scale" if blocks else "k_scale")
        raise ValueError("k_scale and v_scale must both be tensors or both numbers")
    num_pages, P, Hkv, D = shape
    if blocks:
        ksp, kss = _block_scales(k_scale, dtype, shape, "k_scale")
        vsp, vss = _block_scales(v_scale, dtype, shape, "v_scale")
        return (kp, vp, ksp, vsp, code, Hkv, D, P, num_pages, 1.0, 1.0, kst[0], kst[1], kst[2], vst[0], vst[1], vst[2],
                kss[0], kss[1], vss[0], vss[1]), True
    ks, vs = _whole_scale(k_scale, dtype, "k_scale"), _whole_scale(v_scale, dtype, "v_scale")
    return (kp, vp, 0, 0, code, Hkv, D, P, num_pages, ks, vs, kst[0], kst[1], kst[2], vst[0], vst[1], vst[2],
            0, 0, 0, 0), False


def key_cache_fields(k_cache, k_scale):
    """``cache_fields`` of a call that reads K only."""
    code, shape, kp, kst = _cache_layout(k_cache, "k_cache")
    blocks = isinstance(k_scale, torch.Tensor)
    ksp, kss, ks = 0, (0, 0), 1.0
    if blocks:
        ksp, kss = _block_scales(k_scale, k_cache.dtype, shape, "k_scale")
    else:
        ks = _whole_scale(k_scale, k_cache.dtype, "k_scale")
    num_pages, P, Hkv, D = shape
    return (kp, 0, ksp, 0, code, Hkv, D, P, num_pages, ks, 1.0, kst[0], kst[1], kst[2], 0, 0, 0, kss[0], kss[1], 0, 0), blocks


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
    if k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16:
        raise ValueError("append expects bf16 tokens")
    cache, blocks = cache_fields(k_cache, v_cache, k_scale, v_scale)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[2:] != k_cache.shape[2:]:
        raise ValueError("K and V must be [B, N, Hkv, D] matching the caches")
    B, N = shape[0], shape[1]
    pages, table_stride = check_table(block_table, B, "block_table")
    check_lens(seqlens, B, "seqlens")
    written = (k_cache, v_cache)
    if blocks:
        written = (k_cache, v_cache, k_scale, v_scale)
    elif not (k_scale > 0 and v_scale > 0):
        raise ValueError("k_scale and v_scale must be positive")
    new = 0
    if new_lens is not None:
        check_lens(new_lens, B, "new_lens")
        new = new_lens.data_ptr()
    _check_written(*written)
    dev = check_device(k, v, block_table, seqlens, *written)
    if new_lens is not None:
        check_device(k, new_lens)
    kp, vp, ks, vs = k.data_ptr(), v.data_ptr(), k.stride(), v.stride()
    if kp & 15 or vp & 15 or ks[3] != 1 or vs[3] != 1 or (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 7:
        k, v = _prep(k), _prep(v)
        kp, vp, ks, vs = k.data_ptr(), v.data_ptr(), k.stride(), v.stride()
    packed = _lib.pack_kv_append.bytes(
        *cache, kp, vp, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], block_table.data_ptr(),
        table_stride, seqlens.data_ptr(), new, B, N, pages)
    launch(_lib.lib().fgqa_kv_append, packed, dev, "fgqa_kv_append")
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
    if q.dtype is not torch.bfloat16 or q.dim() != 3:
        raise ValueError("expected a bf16 query [B, Hq, D]")
    cache, blocks = key_cache_fields(k_cache, k_scale)
    B, Hq, D = q.shape
    _, page_size, Hkv, _ = k_cache.shape
    if D != 128:
        raise ValueError("the cache's head_dim must match Q")
    if Hq < 1 or Hq % Hkv != 0:
        raise ValueError("Query heads must be divisible by KV heads")
    if lse.dtype is not torch.float32 or lse.shape != (B, Hq) or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 [B, Hq] tensor")
    W, wst = _check_weights(weights, B, Hkv, "weights")
    pages, table_stride = check_table(block_table, B, "block_table")
    check_lens(seqlens, B, "seqlens")
    tokens = pages * page_size
    max_seqlen = min(tokens, W) if max_seqlen is None else check_max_seqlen(max_seqlen, tokens)
    if W < max_seqlen:
        raise ValueError("weights must hold max_seqlen tokens")
    _check_written(weights)
    dev = check_device(q, k_cache, lse, block_table, seqlens, weights)
    if blocks:
        check_device(q, k_scale)
    q = _prep(q)
    qst = q.stride()
    packed = _lib.pack_kv_weights.bytes(
        *cache, q.data_ptr(), lse.data_ptr(), weights.data_ptr(), qst[0], qst[1], wst[0], wst[1], block_table.data_ptr(),
        table_stride, seqlens.data_ptr(), B, max_seqlen, Hq, _SCALE if scale is None else float(scale))
    launch(_lib.lib().fgqa_kv_weights, packed, dev, "fgqa_kv_weights")
    return weights


_SCALE = 1.0 / math.sqrt(128)


def _check_weights(w, B, Hkv, name):
    """(tokens of a row, strides) of weights."""
    shape, st = w.shape, w.stride()
    if w.dtype is not torch.float32 or len(shape) != 3 or shape[0] != B or shape[1] != Hkv \
            or (st[2] != 1 and shape[2] > 1 and w.numel() > 1):
        raise ValueError(f"{name} must be an fp32 [B, Hkv, W] tensor with contiguous rows")
    return shape[2], st


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
    cache, blocks = cache_fields(k_cache, v_cache, k_scale, v_scale)
    _, page_size, Hkv, _ = k_cache.shape
    budget, recent = int(budget), int(recent)
    if not 1 <= budget < 1 << 31 or recent < 0:
        raise ValueError("budget must be positive (and below 2^31) and recent not negative")
    recent = min(recent, budget)
    if seqlens.dim() != 1:
        raise ValueError("seqlens must be a contiguous int32 [B] tensor")
    B = seqlens.shape[0]
    check_lens(seqlens, B, "seqlens")
    W, wst = _check_weights(weights, B, Hkv, "weights")
    pages, table_stride = check_table(block_table, B, "block_table")
    new_pages, new_stride = check_table(new_block_table, B, "new_block_table")
    tokens = pages * page_size
    max_seqlen = min(tokens, W) if max_seqlen is None else check_max_seqlen(max_seqlen, tokens)
    if W < max_seqlen:
        raise ValueError("weights must hold max_seqlen tokens")
    if new_pages * page_size < min(budget, max_seqlen):
        raise ValueError("new_block_table must have pages for min(budget, max_seqlen) tokens")
    given = []
    if new_seqlens is not None:
        check_lens(new_seqlens, B, "new_seqlens")
        given.append(new_seqlens)
    if new_weights is not None:
        if _check_weights(new_weights, B, Hkv, "new_weights")[0] != W:
            raise ValueError("new_weights must have weights' shape")
        _check_written(new_weights)
        given.append(new_weights)
    if kept is not None:
        if kept.dtype is not torch.int32 or kept.shape != (B, Hkv, budget) or not kept.is_contiguous():
            raise ValueError("kept must be a contiguous int32 [B, Hkv, budget] tensor")
        given.append(kept)
    for i, t in enumerate(given):
        if any(_meet(t, x) for x in (*given[:i], weights, seqlens, block_table, new_block_table)):
            raise ValueError("new_seqlens, new_weights and kept must be apart from each other and from the inputs")
    written = (k_cache, v_cache, k_scale, v_scale) if blocks else (k_cache, v_cache)
    _check_written(*written)
    dev = check_device(weights, block_table, seqlens, new_block_table, *written, *given)
    if new_seqlens is None:
        new_seqlens = torch.empty_like(seqlens)
    if new_weights is None:
        new_weights = torch.empty((B, Hkv, W), device=weights.device, dtype=torch.float32)
    if kept is None:
        kept = torch.empty((B, Hkv, budget), device=weights.device, dtype=torch.int32)
    nst = new_weights.stride()
    packed = _lib.pack_kv_evict.bytes(
        *cache, weights.data_ptr(), new_weights.data_ptr(), wst[0], wst[1], nst[0], nst[1], block_table.data_ptr(),
        new_block_table.data_ptr(), table_stride, new_stride, seqlens.data_ptr(), new_seqlens.data_ptr(), kept.data_ptr(),
        B, max_seqlen, W, budget, recent)
    launch(_lib.lib().fgqa_kv_evict, packed, dev, "fgqa_kv_evict")
    return new_seqlens, new_weights, kept
