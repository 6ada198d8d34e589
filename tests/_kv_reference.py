"""The paged KV cache's operators from their definitions, in float64 on the CPU.

Caches are held as decoded codes (float64; bf16 values themselves) with their
block scales apart, so results compare exactly: scales and codes are decided by
roundings of numbers that float64 holds exactly."""
import math

import numpy as np
import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def numbers(cache):
    """Decoded codes of a cache tensor, float64 on the CPU."""
    return cache.detach().cpu().to(torch.float32).double().numpy()


def round_e4m3(y):
    """To the nearest e4m3 value, ties to even, saturated."""
    y = np.clip(y, -448.0, 448.0)
    a = np.abs(y)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(a > 0, a, 1.0)))
    # (log2 next to a power of two)
    e = np.where(np.exp2(e) > a, e - 1, e)
    e = np.where(np.exp2(e + 1) <= a, e + 1, e)
    step = np.exp2(np.maximum(e, -6.0) - 3.0)
    return np.rint(y / step) * step


def round_code(y, dtype):
    if dtype == "e4m3":
        return round_e4m3(y)
    return np.clip(np.rint(np.where(np.isnan(y), 0.0, y)), -127.0, 127.0)


def power_scale(amax, dtype):
    s = 2.0 ** -126
    while s * QMAX[dtype] < amax:
        s *= 2.0
    return s


def finite_max(x):
    x = np.abs(x[np.isfinite(x)])
    return float(x.max()) if x.size else 0.0


def append(cache, scales, dtype, x, table, lens, news, whole=1.0):
    """Writes rows x [B, N, H, D] into `cache` [pages, P, H, D] / `scales` in place."""
    pages, P, H, _ = cache.shape
    for b in range(len(lens)):
        a = max(int(lens[b]), 0)
        n = min(max(int(news[b]), 0), x.shape[1])
        end = min(a + n, table.shape[1] * P)
        for j in range(a // P, -(-end // P) if end > a else a // P):
            page = int(table[b, j])
            if not 0 <= page < pages:
                continue
            t0, t1 = max(a, j * P), min(end, (j + 1) * P)
            s0, s1 = t0 - j * P, t1 - j * P
            rows = x[b, t0 - a:t1 - a]
            if dtype == "bf16":
                cache[page, s0:s1] = rows
                continue
            for h in range(H):
                if scales is None:
                    cache[page, s0:s1, h] = round_code(quotient(rows[:, h], whole), dtype)
                    continue
                s = power_scale(finite_max(rows[:, h]), dtype)
                if s0 > 0:
                    old = float(scales[page, h])
                    if s > old:
                        held = (cache[page, :s0, h] * old).astype(np.float32).astype(np.float64)
                        cache[page, :s0, h] = round_code(held / s, dtype)
                    else:
                        s = old
                cache[page, s0:s1, h] = round_code(quotient(rows[:, h], s), dtype)
                scales[page, h] = s


def quotient(x, s):
    """x / s as fp32 division gives it (exact in the definition's powers of two)."""
    with np.errstate(invalid="ignore", over="ignore"):
        return (x.astype(np.float32) / np.float32(s)).astype(np.float64)


def gather(cache, scales, table, b, n, h, whole=1.0):
    """Sequence b's first n values of head h, [n, D]."""
    P = cache.shape[1]
    ids = np.arange(n)
    pages = np.clip(table[b][ids // P], 0, cache.shape[0] - 1)
    x = cache[pages, ids % P, h]
    return x * (scales[pages, h][:, None] if scales is not None else whole)


def scores(q, k, scale):
    """(scores [G, n], the largest sum of |products| behind one)."""
    return q @ k.T * scale, float((np.abs(q) @ np.abs(k).T).max(initial=0.0)) * abs(scale)


def decode(q, kc, ks, vc, vs, table, lens, scale):
    """(o, lse, |o|'s sum of absolute terms, bound on a score's absolute error)."""
    B, Hq, D = q.shape
    H = kc.shape[2]
    G = Hq // H
    o, mass = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    lse, err = np.full((B, Hq), -np.inf), np.zeros((B, Hq))
    for b in range(B):
        n = int(lens[b])
        for h in range(H if n > 0 else 0):
            k, v = gather(kc, ks, table, b, n, h), gather(vc, vs, table, b, n, h)
            r = slice(h * G, (h + 1) * G)
            s, size = scores(q[b, r], k, scale)
            m = s.max(axis=1, keepdims=True)
            p = np.exp(s - m)
            total = p.sum(axis=1, keepdims=True)
            o[b, r], mass[b, r] = p @ v / total, p @ np.abs(v) / total
            lse[b, r] = (m + np.log(total))[:, 0]
            err[b, r] = score_error(size, np.abs(s).max())
    return o, lse, mass, err


def score_error(size, largest):
    """Bound on the absolute error of an fp32 score and of what its exponential
    makes of it: 128 exact products summed in fp32 in any order (127 roundings of
    partial sums at most `size` large), the scales' two roundings and the change
    to base 2 with a subtraction (4 roundings of numbers up to 1.45 times twice the
    largest score), at half a step of 2^-23 each."""
    return 2.0 ** -24 * (129.0 * size + 12.0 * largest + 8.0)


def weights(q, kc, ks, table, lens, lse, scale, W, whole=1.0):
    """(what is added to the weights, a bound on its error)."""
    B, Hq, _ = q.shape
    H = kc.shape[2]
    G = Hq // H
    w, tol = np.zeros((B, H, W)), np.zeros((B, H, W))
    for b in range(B):
        n = int(lens[b])
        for h in range(H if n > 0 else 0):
            r = slice(h * G, (h + 1) * G)
            s, size = scores(q[b, r], gather(kc, ks, table, b, n, h, whole), scale)
            p = np.exp(s - lse[b, r][:, None])
            w[b, h, :n] = p.sum(axis=0)
            e = score_error(size, max(np.abs(s).max(), np.abs(lse[b, r]).max()))
            # the exponential's error, exp2's own ulp, 16 additions
            tol[b, h, :n] = p.sum(axis=0) * (1.01 * e + 2.0 ** -24 * 20)
    return w, tol


def keep(w, n, budget, recent):
    """Indices kept of a row of n weights."""
    if n <= budget:
        return np.arange(n)
    near = min(recent, budget)
    order = sorted(range(n - near), key=lambda i: (-math.inf if math.isnan(w[i]) else -w[i], not math.isnan(w[i]), i))
    return np.array(sorted(order[:budget - near]) + list(range(n - near, n)), dtype=np.int64)


def evict(kc, ks, vc, vs, dtype, table, new_table, lens, w, budget, recent, whole=None):
    """Moves kept tokens inside the caches (in place); (new_lens, new_w, kept)."""
    B, H, W = w.shape
    pages, P = kc.shape[:2]
    new_lens = np.minimum(lens, budget)
    new_w, kept = np.zeros_like(w), np.full((B, H, budget), -1, dtype=np.int64)
    old = [x if x is None else x.copy() for x in (kc, ks, vc, vs)]
    for b in range(B):
        n, c = int(lens[b]), int(new_lens[b])
        for h in range(H):
            ids = keep(w[b, h, :n], n, budget, recent)
            kept[b, h, :c] = ids
            new_w[b, h, :c] = w[b, h, ids]
            for j in range(-(-c // P)):
                page = int(new_table[b, j])
                if not 0 <= page < pages:
                    continue
                part = ids[j * P:(j + 1) * P]
                src = np.clip(table[b][part // P], 0, pages - 1)
                for cache, scales, oc, osc in ((kc, ks, old[0], old[1]), (vc, vs, old[2], old[3])):
                    rows = oc[src, part % P, h]
                    if scales is not None:
                        rows = (rows * osc[src, h][:, None]).astype(np.float32).astype(np.float64)
                        s = power_scale(finite_max(rows), dtype)
                        rows = round_code(rows / s, dtype)
                        scales[page, h] = s
                    cache[page, :len(part), h] = rows
    return new_lens, new_w, kept
