"""The decode of sequences that begin alike over caches whose slots lie 2^32 bytes apart and more (a cache
with its slots outermost, as [page_size, num_pages, Hkv, D] memory seen as [num_pages, page_size, Hkv, D])."""
import pytest

from tests.test_gpu_kv_shared import Case

pytestmark = pytest.mark.gpu


def far_slots(torch, t):
    """t's values with 2^32 bytes and all pages' rows of one slot from a slot to the next; zeros elsewhere."""
    n, P, H, D = t.shape
    step = (1 << 32) // t.element_size() + n * H * D
    raw = torch.zeros(((P - 1) * step + n * H * D) * t.element_size(), dtype=torch.uint8, device=t.device).view(t.dtype)
    far = raw.as_strided(t.shape, (H * D, step, D, 1))
    for slot in range(P):
        far[:, slot].view(torch.uint8).copy_(t[:, slot].contiguous().view(torch.uint8))
    return far


@pytest.mark.parametrize("dtype,scales,P", [("bf16", None, 2), ("bf16", None, 4), ("e4m3", "whole", 2), ("e4m3", "blocks", 4),
                                            ("int8", "blocks", 2)])
def test_slots_past_32_bits(cuda, dtype, scales, P):
    import torch
    print(dtype, scales, P, flush=True)
    c = Case(torch, cuda, dtype, 8, 2, P, [300], [[9, 40, 1]], [77], scales=scales)
    c.check(*c.run())
    c.cache = [far_slots(torch, t) for t in c.cache]
    assert all(t.stride(1) * t.element_size() >= 1 << 32 for t in c.cache)
    out, lse = c.run()
    c.check(out, lse)
