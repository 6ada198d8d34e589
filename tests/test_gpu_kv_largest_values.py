"""Blocks that hold the largest bf16 numbers: a code times its scale can pass fp32's
largest number (the largest bf16 number rounds up to 2^128), and such blocks are
moved and grown like all others."""
import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import Cache, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


def _scale(amax, dtype):
    return max(ref.power_scale(amax, dtype), 2.0 ** -126)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [4, 16, 64, 512])
def test_evict_blocks_of_the_largest_values(cuda, P, dtype):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    print(f"largest values P={P} {dtype}", flush=True)
    rng = np.random.default_rng(4000 + P)
    n, budget, H = 600, 200, 2
    width, nwidth = -(-n // P), -(-budget // P)
    pages = width + nwidth
    c = Cache(cuda, rng, dtype, pages, P, H)
    both = _table(rng, 1, pages, pages)
    table, new = both[:, :width], both[:, width:]
    top = float(torch.finfo(torch.bfloat16).max)
    k = _x(rng, 1, n, H, 128)
    k[0, 30:40], k[0, 300:310, 1], k[0, 595:] = -top, top, -top     # whole rows
    k[0, 100, 0, 7] = top                                            # one value among ordinary ones
    lens = _i32(cuda, [n])
    fg.append_kv_paged(k.to(cuda), (-k).to(cuda), c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, [0]), **c.scales)
    torch.cuda.synchronize()
    for i, x in enumerate((k, -k)):
        ref.append(c.n[i], c.sn[i], dtype, x.float().numpy().astype(np.float64), table, [0], [n])
    c.check("append")
    w = rng.exponential(size=(1, H, n)).astype(np.float32)
    w[:, :, [30, 35, 100, 300]] = 1e9
    _, _, kept = fg.evict_kv_paged(c.t[0], c.t[1], _i32(cuda, table), lens, torch.from_numpy(w).to(cuda), _i32(cuda, new),
                                   budget=budget, recent=8, **c.scales)
    torch.cuda.synchronize()
    for i in range(2):
        codes, scales = c.n[i].copy(), c.sn[i].copy()
        for h in range(H):
            ids = ref.keep(w[0, h], n, budget, 8)
            assert np.array_equal(kept[0, h].cpu().numpy(), ids)
            for j in range(nwidth):
                part = ids[j * P:(j + 1) * P]
                rows = c.n[i][table[0][part // P], part % P, h] * c.sn[i][table[0][part // P], h][:, None]
                s = _scale(np.abs(rows).max(), dtype)
                codes[new[0, j], :len(part), h] = ref.round_code(rows / s, dtype)
                scales[new[0, j], h] = s
        c.n[i], c.sn[i] = codes, scales
    c.check("evict")


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [16, 512])
def test_append_grows_a_block_near_the_end_of_the_range(cuda, P, dtype):
    """Old codes under a scale that is no power of two, whose products pass fp32's
    largest number, rounded again to the scale of the largest bf16 number."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    rng = np.random.default_rng(4100 + P)
    c = Cache(cuda, rng, dtype, 3, P, 1)
    qmax = int(ref.QMAX[dtype])
    for i in range(2):
        c.t[i].view(torch.uint8)[:] = torch.tensor([float(qmax)]).to(ref.DTYPES[dtype]).view(torch.uint8).to(cuda)
        c.s[i].fill_(1.9 * 2.0 ** (119 if dtype == "e4m3" else 121))
        c.n[i][:] = qmax
        c.sn[i] = c.s[i].cpu().double().numpy()
    top = float(torch.finfo(torch.bfloat16).max)
    k = torch.full((1, 3, 1, 128), top, dtype=torch.bfloat16)
    table = np.array([[1]], dtype=np.int32)
    fg.append_kv_paged(k.to(cuda), k.to(cuda), c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, [9]), **c.scales)
    torch.cuda.synchronize()
    s = _scale(top, dtype)
    for i in range(2):
        c.n[i][1, :9] = ref.round_code(c.n[i][1, :9] * c.sn[i][1, 0] / s, dtype)
        c.n[i][1, 9:12] = ref.round_code(np.full((3, 1, 128), top) / s, dtype)
        c.sn[i][1] = s
    c.check("grown")
