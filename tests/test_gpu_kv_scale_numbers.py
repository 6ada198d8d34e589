"""GPU tests: one scale for a whole e4m3 cache as a tensor of one element, on the host or
the GPU, gives what the number gives."""
import numpy as np
import pytest

from tests.test_gpu_kv_cache import Cache, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["cpu", "cuda", "double"])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_tensors_of_one_element(cuda, shape, where):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    P, H = 16, 2

    def run(k_scale, v_scale):
        rng = np.random.default_rng(5000)
        c = Cache(cuda, rng, "e4m3", 30, P, H, scales=False)
        both = _table(rng, 2, 15, 30)
        table, new = _i32(cuda, both[:, :10]), _i32(cuda, both[:, 10:])
        lens, after = _i32(cuda, [100, 37]), _i32(cuda, [105, 42])
        x = _x(rng, 2, 5, H, 128).to(cuda)
        q = _x(rng, 2, 8, 128).to(cuda)
        lse, w = torch.empty((2, 8), device=cuda), torch.zeros((2, H, 160), device=cuda)
        fg.append_kv_paged(x, x, c.t[0], c.t[1], table, lens, k_scale=k_scale, v_scale=v_scale)
        o = fg.decode_flash_gqa_paged(q, c.t[0], c.t[1], table, after, lse=lse, k_scale=k_scale, v_scale=v_scale)
        fg.accumulate_kv_weights_paged(q, c.t[0], lse, table, after, w, k_scale=k_scale)
        out = fg.evict_kv_paged(c.t[0], c.t[1], table, after, w, new, 70, 8, k_scale=k_scale, v_scale=v_scale)
        torch.cuda.synchronize()
        return [t.view(torch.uint8) for t in c.t] + [o, lse, w, *out]

    def one(x):
        t = torch.full(shape, x, dtype=torch.float64 if where == "double" else torch.float32)
        return t.to(cuda) if where == "cuda" else t

    want = run(0.25, 0.5)
    for a, b in zip(want, run(one(0.25), one(0.5))):
        assert torch.equal(a, b)
    for a, b in zip(want, run(0.25, one(0.5))):
        assert torch.equal(a, b)
