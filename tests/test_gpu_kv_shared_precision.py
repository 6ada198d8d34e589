"""The decode of sequences that begin alike over caches with block scales holds P times V's scale over shared tokens to
more bits than one bf16 number has: tokens of two score levels whose values cancel, so that every token of a
level is rounded alike and the output is far smaller than its terms."""
import math

import numpy as np
import pytest

from tests.test_gpu_kv_shared import Case, D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [1, 8, 16, 64])
def test_levels_that_cancel(cuda, P, dtype):
    import torch
    print(dtype, P, flush=True)
    c = Case(torch, cuda, dtype, 16, 2, P, [256], [[1, 2, 3]], [], scales="blocks")
    code = lambda x: torch.tensor([float(x)]).to(c.cache[0].dtype).view(torch.uint8).to(cuda)
    raw = [t.view(torch.uint8) for t in c.cache]
    for t in raw:
        t.zero_()
    for s in ("k_scale", "v_scale"):
        c.kw[s].fill_(2.0 ** -5)
    # even tokens: K 1, V 80 / 32; odd ones: K 0.75, V -112 / 32, whose weight is e^(-0.25 q / sqrt(128)), 80 / 112 or so
    for t in range(256):
        page, slot = int(c.table[0, t // P]), t % P
        raw[0][page, slot, :, 0] = code(24 if t % 2 else 32)
        raw[1][page, slot] = code(-112 if t % 2 else 80)
    c.q.zero_()
    c.q[:, :, 0] = 15 + torch.arange(16, device=cuda) / 8
    out, _ = c.run()
    q, table = c.q.double().cpu().numpy(), c.table.cpu().numpy()
    k, v = (x.cpu().double().numpy() * 2.0 ** -5 for x in c.cache)
    out = out.double().cpu().numpy()
    for b, n in enumerate(c.lens):
        pages = table[b, :-(-n // P)]
        kk, vv = (x[pages].reshape(-1, 2, D)[:n] for x in (k, v))
        for h in range(2):
            rows = slice(8 * h, 8 * h + 8)
            s = q[b, rows] @ kk[:, h].T / math.sqrt(D)
            # fp32 products, sums and exponents of the scores
            e = 2.0 ** -17 * (np.abs(q[b, rows]) @ np.abs(kk[:, h]).T) / math.sqrt(D)
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            want = p @ vv[:, h]
            # P sV in two bf16 numbers: half a step of 2^-7, and half of one more: 2^-16.  fp32 sums of the
            # numerator and the denominator: 2^-24 a token, 40 for the exponent, the rescaling and the merge
            moved = (p * (2.0 ** -16 + e + (p * e).sum(axis=1, keepdims=True) + 2.0 ** -23 * (n + 40))) @ np.abs(vv[:, h])
            d = np.abs(out[b, rows] - want)
            bound = 2.0 ** -8 * np.abs(want) + moved
            assert (d <= bound).all(), (b, h, float((d / bound).max()), float(np.abs(want).max()), float(bound.max()))
