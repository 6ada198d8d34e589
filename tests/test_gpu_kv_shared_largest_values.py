"""The decode of sequences that begin alike over values near bf16's largest, with a score that rises on the way: weights
held above 1 for a while would make sums, or a weight times its block's scale, infinite where the
decode of each sequence on its own gives numbers."""
import math

import numpy as np
import pytest

from tests.test_gpu_kv_shared import Case

pytestmark = pytest.mark.gpu

KINDS = [("bf16", None), ("e4m3", "whole"), ("e4m3", "blocks"), ("int8", "blocks")]


def _case(torch, cuda, dtype, scales, P):
    """Keys whose scores lie near 0, but for tokens 200 and 400 of the 512 shared ones: 4 (or what the codes hold) times
    16 / sqrt(128) above, 5 to 8 powers of 2."""
    c = Case(torch, cuda, dtype, 8, 2, P, [512], [[40, 7, 30]], [90], scales=scales)
    c.q *= 0.25
    c.q[:, :, 0] = 16
    k, v = c.cache[0], c.values[0]
    raw = torch.uint8 if k.element_size() == 1 else torch.int16
    k.view(raw)[..., 0] = 0
    v[..., 0] = 0
    for t in (200, 400):
        page, slot = int(c.table[0, t // P]), t % P
        s = c.kw.get("k_scale", 1.0)
        for h in range(2):
            step = s if isinstance(s, float) else float(s[page, h])
            top = {"bf16": 4.0, "e4m3": 448.0, "int8": 127.0}[dtype]
            one = torch.tensor([min(4.0 / step, top)]).to(k.dtype)
            k.view(raw)[page, slot, h, 0] = int(one.view(raw))
            v[page, slot, h, 0] = float(one.double()) * step
    return c


@pytest.mark.parametrize("dtype,scales", KINDS)
@pytest.mark.parametrize("P", [1, 16, 64])
def test_sums_of_large_values(cuda, dtype, scales, P):
    """Values up to 2^124: weights of at most 1 leave sums below 2^128, those of 2^5 to 2^8 do not."""
    import torch
    print(dtype, scales, P, flush=True)
    c = _case(torch, cuda, dtype, scales, P)
    up = 2.0 ** (123 - math.floor(math.log2(max(np.abs(np.nan_to_num(c.values[1])).max(), 1e-30))))
    c.values[1] *= up
    if dtype == "bf16":
        c.cache[1] *= up
    else:
        c.kw["v_scale"] *= up
    out, lse = c.run()
    c.check(out, lse)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [1, 16, 64])
def test_scales_of_large_blocks(cuda, dtype, P):
    """Blocks of the largest scale that is written, nearly all codes 0: their products stay 0."""
    import torch
    print(dtype, P, flush=True)
    c = _case(torch, cuda, dtype, "blocks", P)
    top = 2.0 ** (120 if dtype == "e4m3" else 122)
    v, kept = c.cache[1].view(torch.uint8), c.values[1]
    pages = c.table[0, :512 // P].long()
    one = torch.tensor([1.0]).to(c.cache[1].dtype).view(torch.uint8).to(cuda)
    v[pages] = 0
    v[pages[::3], 0, :, 5] = one
    kept[pages.cpu().numpy()] = 0
    kept[pages[::3].cpu().numpy(), 0, :, 5] = top
    c.kw["v_scale"][pages] = top
    out, lse = c.run()
    c.check(out, lse)
