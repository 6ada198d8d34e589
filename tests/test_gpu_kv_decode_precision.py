"""The block-scaled decode holds P to more bits than an fp16 number has: values
that cancel show it, whose sum is far smaller than its terms."""
import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import Cache, _for_teams, _i32, _table, _torch, _x
from tests.test_gpu_kv_decode_far_scales import exact_with_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["whole", "splits", "teams"])
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [4, 8, 16, 64])
def test_values_that_cancel(cuda, P, dtype, form):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    print(f"cancelling values P={P} {dtype} {form}", flush=True)
    rng = np.random.default_rng(2200 + P)
    lens = [192, 2, 64]
    width = -(-192 // P)
    c = Cache(cuda, rng, dtype, 3 * width, P, 2)
    table = _table(rng, 3, width, 3 * width)
    # tokens 2i and 2i + 1: opposite values (a code's top bit is its sign in e4m3; int8
    # is negated), under one scale; scores near 0, so that the P's differ little
    raw = c.t[1].view(torch.uint8)
    c.s[1].fill_(0.5)
    for b, n in enumerate(lens):
        for t in range(0, n, 2):
            row = raw[int(table[b, t // P]), t % P]
            other = row ^ 0x80 if dtype == "e4m3" else (-row.view(torch.int8)).view(torch.uint8)
            raw[int(table[b, (t + 1) // P]), (t + 1) % P] = other
    c.n[1] = ref.numbers(c.t[1])
    c.sn[1][:] = 0.5
    q = _x(rng, 3, 6, 128) * 2.0 ** -9
    # (P sV in two fp16 numbers: half a step of 22 bits, and half of one more)
    o, tol = exact_with_bound(q.float().numpy().astype(np.float64), c, table, lens, p_error=2.0 ** -21)
    of = _for_teams(cuda, table, P, 2) if form == "teams" else table
    got = fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, of), _i32(cuda, lens),
                                    split_tokens=128 if form == "splits" else 0, **c.scales)
    torch.cuda.synchronize()
    got = got.float().cpu().double().numpy()
    bad = np.abs(got - o) > tol + 2.0 ** -8 * np.abs(o)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, by {(np.abs(got - o) / tol).max():.1f} times the bound"
