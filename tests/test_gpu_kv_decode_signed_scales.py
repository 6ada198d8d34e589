"""Block-scaled decode: a block under a scale of the other sign, with its codes negated,
gives the same outputs."""
import numpy as np
import pytest

from tests.test_gpu_kv_cache import Cache, _for_teams, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [4, 16, 64])
def test_negative_scales(cuda, P):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    rng = np.random.default_rng(8000 + P)
    width = -(-300 // P)
    c = Cache(cuda, rng, "int8", width, P, 2)
    table, lens = _table(rng, 1, width, width), _i32(cuda, [300])
    q = _x(rng, 1, 8, 128).to(cuda)
    for t in (_i32(cuda, table), _i32(cuda, _for_teams(cuda, table, P, 2))):
        want = fg.decode_flash_gqa_paged(q, c.t[0], c.t[1], t, lens, **c.scales)
        flip = torch.from_numpy(rng.integers(0, 2, size=(width, 2)) * 2 - 1).to(cuda)
        caches = [(x * flip[:, None, :, None]).to(torch.int8) for x in c.t]
        got = fg.decode_flash_gqa_paged(q, *caches, t, lens, k_scale=c.s[0] * flip, v_scale=c.s[1] * flip)
        torch.cuda.synchronize()
        assert torch.equal(want, got)
