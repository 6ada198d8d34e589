"""The decode of sequences that begin alike over K blocks of the least scale, 2^-126, which the scores' scale takes below
the normal numbers, and queries as far above 1."""
import pytest

from tests.test_gpu_kv_shared import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [1, 16, 64])
def test_least_scales_of_keys(cuda, P, dtype):
    """Scores of some 0.02 (2^112 to 2^114 times codes of 2^-126): not 8 times that, nor 0."""
    import torch
    print(dtype, P, flush=True)
    c = Case(torch, cuda, dtype, 8, 2, P, [512], [[40, 7, 30]], [90])
    c.values[0] *= 1 / c.kw["k_scale"].double().cpu().numpy()[:, None, :, None] * 2.0 ** -126
    c.kw["k_scale"].fill_(2.0 ** -126)
    c.q = (c.q.float() * 2.0 ** (114 if dtype == "int8" else 112)).to(torch.bfloat16)
    out, lse = c.run()
    c.check(out, lse)
