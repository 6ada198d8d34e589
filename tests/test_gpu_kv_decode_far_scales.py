"""Block-scaled decode where a V block of a far larger scale gets next to no
attention: the tokens that get it keep their bits.  Every output row is held to a
bound made of its own terms."""
import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import SCALE, Cache, _for_teams, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


def exact_with_bound(q, c, table, lens, p_error=2.0 ** -11):
    """(o, a bound on the error of O before it is rounded to bf16), each output by
    its own terms p_t sV_t c_t: P sV to half a step of an fp16 number (p_error), or
    2^-39 of the row's largest one where that is more (fp16 subnormals, half a step
    2^-25 at 2^14); fp32 products and sums, numerator and denominator, at half a step of
    2^-23 each, 40 for the exponential, the rescaling and the merges; the scores'
    errors in both."""
    o, lse, mass, err = ref.decode(q, c.n[0], c.sn[0], c.n[1], c.sn[1], table, lens, SCALE)
    G = q.shape[1] // c.n[0].shape[2]
    tol = mass * (p_error + 2.2 * err[..., None] + 2.0 ** -24 * 2 * (max(lens) + 40))
    P = c.n[0].shape[1]
    for b, n in enumerate(lens):
        for h in range(c.n[0].shape[2]):
            r = slice(h * G, (h + 1) * G)
            s = q[b, r] @ ref.gather(c.n[0], c.sn[0], table, b, n, h).T * SCALE
            sv = c.sn[1][table[b][np.arange(n) // P], h]
            codes = ref.gather(c.n[1], None, table, b, n, h)
            w = np.exp(s - lse[b, r][:, None]) * sv
            tol[b, r] += 2.0 ** -39 * w.max(axis=1)[:, None] * np.abs(codes).sum(axis=0)
    return o, tol


@pytest.mark.parametrize("form", ["whole", "splits", "teams"])
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [4, 8, 16, 64])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_a_large_block_without_attention(cuda, place, P, dtype, form):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    print(f"far scales {place} P={P} {dtype} {form}", flush=True)
    rng = np.random.default_rng(2000 + P)
    H, lens = 2, [450, 100]
    width = -(-450 // P)
    c = Cache(cuda, rng, dtype, 2 * width, P, H)
    table = _table(rng, 2, width, 2 * width)
    q = _x(rng, 2, 8, 128) * 0.125
    q[:, :, 0] = 8.0
    code = torch.tensor([-96.0]).to(ref.DTYPES[dtype]).view(torch.uint8).to(cuda)   # -96 in either type
    for cache in (c.t[0], c.t[1]):   # channel 0: no part in the ordinary scores
        cache.view(torch.uint8)[:, :, :, 0] = 0
    for b, n in enumerate(lens):
        last = (n - 1) // P
        page = int(table[b, {"first": 0, "middle": last // 2, "last": last}[place]])
        c.t[0].view(torch.uint8)[page, :, :, 0] = code
        c.s[0][page] = 1.0                      # scores of about -68: P 2^-98
        c.s[1][page] *= 2.0 ** 50
    for i in range(2):
        c.n[i] = ref.numbers(c.t[i])
        c.sn[i] = c.s[i].cpu().double().numpy()
    of = _for_teams(cuda, table, P, H) if form == "teams" else table
    got = fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, of), _i32(cuda, lens),
                                    split_tokens=128 if form == "splits" else 0, **c.scales)
    torch.cuda.synchronize()
    got = got.float().cpu().double().numpy()
    o, tol = exact_with_bound(q.float().numpy().astype(np.float64), c, table, lens)
    bad = np.abs(got - o) > tol + 2.0 ** -8 * np.abs(o)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, {np.abs(got - o).max()} at most of {np.abs(o).max()}"


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [4, 16, 64])
def test_every_row_by_its_own_terms(cuda, P, dtype):
    """V scales over 2^60 in every order, and heads of far smaller values than others."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    rng = np.random.default_rng(2100 + P)
    lens = [500, 77]
    width = -(-500 // P)
    c = Cache(cuda, rng, dtype, 2 * width, P, 2)
    table = _table(rng, 2, width, 2 * width)
    c.sn[1] = np.float32(c.sn[1] * np.exp2(rng.integers(-30, 31, size=c.sn[1].shape)) *
                         rng.uniform(0.5, 1.0, size=c.sn[1].shape)).astype(np.float64)
    c.sn[1][:, 1] *= 2.0 ** -50
    c.s[1] = torch.from_numpy(c.sn[1].astype(np.float32)).to(cuda)
    q = _x(rng, 2, 8, 128)
    o, tol = exact_with_bound(q.float().numpy().astype(np.float64), c, table, lens)
    for t in (table, _for_teams(cuda, table, P, 2)):
        got = fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, t), _i32(cuda, lens), **c.scales)
        torch.cuda.synchronize()
        assert np.all(np.abs(got.float().cpu().double().numpy() - o) <= tol + 2.0 ** -8 * np.abs(o))
