"""Norm and rotation of queries and keys in float64 (numpy), from the formulas."""
import numpy as np


def angles(positions, inv_freq, axes):
    """positions [A, T], inv_freq [R/2] -> float64 [T, R/2]."""
    a = np.zeros(len(inv_freq), dtype=np.int64) if axes is None else np.clip(axes, 0, len(positions) - 1)
    return positions[a].T.astype(np.float64) * inv_freq.astype(np.float64)


def pairs(rotary, interleaved):
    """Indices of the pairs' first and second elements."""
    j = np.arange(rotary // 2)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rotary // 2)


def rotate(x, theta, interleaved, back=False):
    """x [T, H, D] turned by theta [T, R/2] (back: by -theta)."""
    out = x.copy()
    a, b = pairs(2 * theta.shape[1], interleaved)
    c, s = np.cos(theta)[:, None, :], np.sin(theta)[:, None, :] * (-1 if back else 1)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def pair_size(x, rotary, interleaved):
    """|a| + |b| of each element's pair; |x| where there is none."""
    out = np.abs(x)
    a, b = pairs(rotary, interleaved)
    both = out[..., a] + out[..., b]
    out[..., a] = out[..., b] = both
    return out


def forward(x, w, theta, eps, interleaved):
    """(values, bound of the kernel's error but for the last rounding), x [T, H, D] float64.

    In fp32 a sum of D squares in a tree of at most 20 additions, the reciprocal root (2^-22),
    two products, the rotation's two products and sum, and cos and sin off by at most
    2^-22 (the fraction of a turn rounded to 24 bits, 2^-23.3 in radians, and their
    polynomials): 2^-19 of |a| + |b| in all."""
    u = x
    if w is not None:
        u = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * w
    return rotate(u, theta, interleaved), 2.0 ** -19 * pair_size(u, 2 * theta.shape[1], interleaved)


def backward(dy, x, w, theta, eps, interleaved):
    """(dx, its bound, dw, its bound); the bounds count as forward's, the sums' adds with them."""
    g = rotate(dy, theta, interleaved, back=True)
    g_size = pair_size(dy, 2 * theta.shape[1], interleaved)
    if w is None:
        return g, 2.0 ** -19 * g_size, None, None
    r = 1.0 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps)
    u = x * r
    dw = (g * u).sum(axis=(0, 1))
    dw_bound = 2.0 ** -17 * (g_size * np.abs(u)).sum(axis=(0, 1))
    gw = g * w
    dx = r * (gw - u * (gw * u).mean(axis=-1, keepdims=True))
    bound = 2.0 ** -17 * r * (g_size * np.abs(w) + np.abs(u) * (g_size * np.abs(w * u)).mean(axis=-1, keepdims=True))
    return dx, bound, dw, dw_bound
