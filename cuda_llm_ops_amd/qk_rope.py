"""Queries and keys normalised for each head and rotated to their positions, before
any of the attention calls, over the C ABI of include/fgqa_rope.h.

    qk_norm_rope            the forward pass: prompts, training batches, single tokens
    qk_norm_rope_backward   its gradients

No counterpart in the reference.  PyTorch only provides device memory and the
current stream.  Every tensor of a call lives on one device; the call runs on that
device's current stream.
"""
from __future__ import annotations

from .kv_cache import call_native

__all__ = ["qk_norm_rope", "qk_norm_rope_backward"]


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, axes=None, interleaved=False,
                 q_out=None, k_out=None):
    """RMS norm of each query and key head, then the rotation to its position, in one
    pass; returns (q_out, k_out).

    q, k: bf16 [B, S, Hq, D] and [B, S, Hkv, D], or [T, Hq, D] and [T, Hkv, D] (single
    tokens, packed sequences); D a multiple of 16 up to 256; any strides with contiguous
    rows (views of a fused projection; rows that are not 16-byte aligned are copied).
    q_weight, k_weight: [D], bf16 or fp32 (both None: no norm).
    positions: int32 or int64, [B, S], [S] or, of A axes, [A, B, S] ([T] or [A, T]);
    inv_freq: fp32 [R / 2], the rotation's radians for each step of a position, R a
    multiple of 16 up to D; axes: int32 [R / 2], the axis whose position turns each pair
    (None: one axis; values are clamped to the axes there are).  positions and inv_freq
    None: no rotation.

    With u = x * weight / sqrt(mean(x^2) + eps) and theta_j = positions[axes[j]] *
    inv_freq[j], elements (a, b) = (j, j + R / 2), or (2j, 2j + 1) if ``interleaved``, become
    (u_a cos - u_b sin, u_b cos + u_a sin); those from R on are normalised only.  Angles are
    formed in 64 bits, the rest in fp32, with one rounding to bf16.

    q_out, k_out: bf16, as q and k (allocated when None); q_out may be q itself and k_out
    k (the rows are then replaced), else they lie apart."""
    return call_native("rope", q, q, k, positions, inv_freq, q_weight, k_weight, eps, axes, interleaved, q_out, k_out)


def qk_norm_rope_backward(grad_q, grad_k, q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, axes=None,
                          interleaved=False):
    """The gradients of ``qk_norm_rope``: from those of its outputs (bf16, q's and k's
    shapes) returns (of q, of k, of q_weight, of k_weight).

    The other arguments are the forward call's, q and k its inputs (None will do
    without weights: a rotation's gradients do not depend on them).  Those of q and k are bf16;
    those of the weights are fp32 [D], summed over all rows without atomics, or None
    without weights."""
    return call_native("rope_backward", grad_q, grad_q, grad_k, q, k, positions, inv_freq, q_weight, k_weight, eps, axes,
                       interleaved)
