"""GPU tests: tensors that the paged cache's operators write count as changed, so that
autograd refuses a backward pass over a value it saved before."""
import numpy as np
import pytest

from tests.test_gpu_kv_cache import Cache, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


def _case(cuda, dtype="int8"):
    torch = _torch()
    rng = np.random.default_rng(6000)
    c = Cache(cuda, rng, dtype, 30, 16, 2)
    both = _table(rng, 2, 15, 30)
    return (c, _i32(cuda, both[:, :10]), _i32(cuda, both[:, 10:]), _i32(cuda, [100, 37]), _x(rng, 2, 5, 2, 128).to(cuda),
            _x(rng, 2, 8, 128).to(cuda), torch.full((2, 8), 5.0, device=cuda), torch.zeros((2, 2, 160), device=cuda))


def test_versions(cuda):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    c, table, new, lens, x, q, lse, w = _case(cuda)

    def raised(tensors, call):
        before = [t._version for t in tensors]
        call()
        return [t._version > b for t, b in zip(tensors, before)]

    cache = [*c.t, *c.s]
    assert all(raised(cache, lambda: fg.append_kv_paged(x, x, *c.t, table, lens, **c.scales)))
    assert not any(raised([x, table, lens], lambda: fg.append_kv_paged(x, x, *c.t, table, lens, **c.scales)))
    assert raised([w, q, c.t[0]], lambda: fg.accumulate_kv_weights_paged(q, c.t[0], lse, table, lens, w, k_scale=c.s[0])) == \
        [True, False, False]
    nl, nw, kept = torch.empty_like(lens), torch.empty_like(w), torch.empty((2, 2, 70), dtype=torch.int32, device=cuda)
    assert raised([*cache, nl, nw, kept, w, table, lens], lambda: fg.evict_kv_paged(
        *c.t, table, lens, w, new, 70, 8, new_seqlens=nl, new_weights=nw, kept=kept, **c.scales)) == [True] * 7 + [False] * 3
    torch.cuda.synchronize()


def test_a_saved_value_that_changed(cuda):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    c, table, _, lens, _, q, lse, w = _case(cuda)
    a = torch.ones_like(w, requires_grad=True)
    y = (a * w).sum()
    fg.accumulate_kv_weights_paged(q, c.t[0], lse, table, lens, w, k_scale=c.s[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors(cuda):
    """Tensors without a version are written inside and outside of inference mode."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    c, table, _, lens, x, q, lse, _ = _case(cuda)
    with torch.inference_mode():
        w = torch.zeros((2, 2, 160), device=cuda)
        fg.accumulate_kv_weights_paged(q, c.t[0], lse, table, lens, w, k_scale=c.s[0])
        fg.append_kv_paged(x, x, *c.t, table, lens, **c.scales)
        one = w.clone()
    fg.accumulate_kv_weights_paged(q, c.t[0], lse, table, lens, w, k_scale=c.s[0])
    torch.cuda.synchronize()
    assert bool((w[0, :, :100] >= one[0, :, :100]).all())
