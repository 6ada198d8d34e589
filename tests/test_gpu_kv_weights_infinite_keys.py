"""Attention weights over bf16 caches whose keys hold infinities: a token whose
scores are all -inf gets exactly nothing, whatever the number of query heads of a
KV head; one with a score of +inf gets an infinite weight."""
import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import SCALE, Cache, _i32, _table, _torch, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [4, 8, 64])
@pytest.mark.parametrize("G", [1, 3, 7, 16])
def test_infinite_keys(cuda, G, P):
    import cuda_llm_ops_amd as fg
    torch = _torch()
    print(f"infinite keys G={G} P={P}", flush=True)
    rng = np.random.default_rng(1000 + 16 * G + P)
    H, lens, W = 2, [130, 64, 1], 140
    width = -(-130 // P)
    c = Cache(cuda, rng, "bf16", 3 * width, P, H)
    table = _table(rng, 3, width, 3 * width)
    q = _x(rng, 3, G * H, 128)
    q[:, :, 5] = -(q[:, :, 5].abs() + 1)          # channel 5 is negative in every head, 9 positive
    q[:, :, 9] = q[:, :, 9].abs() + 1
    # (sequence, token, head, channel, value, what the token gets)
    put = [(0, 0, 0, 5, np.inf, 0.0), (0, 77, 1, 9, -np.inf, 0.0), (0, 129, 0, 5, np.inf, 0.0),
           (1, 63, 1, 5, np.inf, 0.0), (2, 0, 0, 9, -np.inf, 0.0), (1, 30, 0, 9, np.inf, np.inf)]
    for b, t, h, d, value, _ in put:
        c.t[0][int(table[b, t // P]), t % P, h, d] = value
    lse = torch.from_numpy(rng.uniform(3, 12, size=(3, G * H)).astype(np.float32)).to(cuda)
    start = rng.uniform(0, 1, size=(3, H, W)).astype(np.float32)
    w = torch.from_numpy(start).to(cuda)
    fg.accumulate_kv_weights_paged(q.to(cuda), c.t[0], lse, _i32(cuda, table), _i32(cuda, lens), w, max_seqlen=130)
    torch.cuda.synchronize()
    got = w.cpu().numpy()
    for b, t, h, _, _, gets in put:
        assert got[b, h, t] == np.float32(start[b, h, t] + gets), f"token {t} of sequence {b}: {got[b, h, t]}"
    # all others: as with keys of zeros in the places of the infinite ones
    others = np.ones_like(start, dtype=bool)
    for b, t, h, d, _, _ in put:
        c.n[0][int(table[b, t // P]), t % P, h, d] = 0.0
        others[b, h, t] = False
    add, tol = ref.weights(q.float().numpy().astype(np.float64), c.n[0], None, table, lens, lse.cpu().double().numpy(), SCALE, W)
    # (a made-up LSE can lie far below the scores: sums past fp32's largest number are inf)
    with np.errstate(invalid="ignore"):
        want = start + add
        over = want > float(np.finfo(np.float32).max)
        good = np.where(over, np.isposinf(got), np.abs(got - want) <= tol + 2.0 ** -23 * np.abs(want))
    assert good[others].all()
