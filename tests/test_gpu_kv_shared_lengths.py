"""Shared lengths far past the sequences': what the shortest one has, whole pages of it, is shared."""
import pytest

from tests.test_gpu_kv_shared import Case

pytestmark = pytest.mark.gpu

FAR = (1 << 30, (1 << 31) - 1)


@pytest.mark.parametrize("dtype", ("bf16", "e4m3"))
def test_shared_lengths_past_the_sequences(cuda, dtype):
    import torch
    c = Case(torch, cuda, dtype, 8, 2, 16, [512], [[40, 7, 300, 1, 20, 2]], [90])
    want, want_lse = c.run([0, 6], [512])
    for far in FAR:
        print(dtype, far, flush=True)
        out, lse = c.run([0, 6], [far])
        c.check(out, lse)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_shared_lengths_past_the_sequences_of_many(cuda):
    """More sequences than the decode's workgroups plan for themselves."""
    import torch
    c = Case(torch, cuda, "int8", 4, 2, 16, [256], [[1 + i % 5 for i in range(300)]], [40, 300])
    want, want_lse = c.run([0, 300], [256])
    for far in FAR:
        print(far, flush=True)
        out, lse = c.run([0, 300], [far])
        c.check(out, lse)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
