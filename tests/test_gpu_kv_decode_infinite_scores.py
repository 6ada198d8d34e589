"""Block-scaled decode over e4m3 codes: keys whose scores overflow to -inf get nothing,
wherever they lie, and keys that are NaN make their heads NaN."""
import math

import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import Cache, _for_teams, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["whole", "splits", "teams"])
@pytest.mark.parametrize("P", [4, 16, 64])
def test_minus_infinity(cuda, P, form):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    print(f"-inf scores P={P} {form}", flush=True)
    rng = np.random.default_rng(7000 + P)
    width = -(-300 // P)
    c = Cache(cuda, rng, "e4m3", 2 * width, P, 1)
    table, lens = _table(rng, 2, width, 2 * width), [300, 40]
    alive = np.zeros(300, bool)
    alive[140:150] = alive[299] = True
    # 3e38 * -1 * 64 / sqrt(128) is past fp32's range; the alive keys' products are 0
    raw = c.t[0].view(torch.uint8)
    raw[:, :, 0, 7] = 0xb8   # -1
    for t in np.flatnonzero(alive):
        raw[int(table[0, t // P]), t % P, 0, 7] = 0
    c.s[0].fill_(64.0)
    q = _x(rng, 2, 2, 128)
    q[:, 0, :] = 0.0
    q[:, 0, 7] = 3e38
    lse = torch.empty((2, 2), device=cuda)
    of = _for_teams(cuda, table, P, 1) if form == "teams" else table
    o = fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, of), _i32(cuda, lens), lse=lse,
                                  split_tokens=128 if form == "splits" else 0, **c.scales)
    torch.cuda.synchronize()
    rows = ref.gather(c.n[1], c.sn[1], table, 0, 300, 0)[alive]
    got = o[0, 0].float().cpu().double().numpy()
    # equal P's of 1; sums of 11 terms and two products in fp32, O to bf16
    assert np.all(np.abs(got - rows.mean(axis=0)) <= 2.0 ** -8 * np.abs(rows.mean(axis=0)) + 2.0 ** -20 * np.abs(rows).mean(axis=0))
    assert abs(float(lse[0, 0]) - math.log(11)) <= 2.0 ** -21
    assert bool(o[1, 0].isnan().all())           # no key of row 1 is alive


@pytest.mark.parametrize("form", ["whole", "splits", "teams"])
@pytest.mark.parametrize("place", [0, 150, 299])
def test_nan_codes(cuda, place, form):
    """A NaN key: its head's outputs and LSE are NaN, other heads' are not.  A NaN among
    the values: its column."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    rng = np.random.default_rng(7100)
    P, width = 16, 19
    c = Cache(cuda, rng, "e4m3", width, P, 3)
    table = _table(rng, 1, width, width)
    page = int(table[0, place // P])
    c.t[0].view(torch.uint8)[page, place % P, 0, 3] = 0x7f
    c.t[1].view(torch.uint8)[page, place % P, 1, 100] = 0xff
    of = _for_teams(cuda, table, P, 3) if form == "teams" else table
    lse = torch.empty((1, 6), device=cuda)
    o = fg.decode_flash_gqa_paged(_x(rng, 1, 6, 128).to(cuda), c.t[0], c.t[1], _i32(cuda, of), _i32(cuda, [300]), lse=lse,
                                  split_tokens=128 if form == "splits" else 0, **c.scales)
    torch.cuda.synchronize()
    nan = o.isnan()[0].cpu()
    assert bool(nan[:2].all()) and not nan[4:].any()
    assert bool(nan[2:4, 100].all()) and int(nan[2:4].sum()) == 2
    assert lse.isnan()[0].tolist() == [True, True, False, False, False, False]
