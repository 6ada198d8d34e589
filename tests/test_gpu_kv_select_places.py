"""Eviction of rows that several workgroups share: nearly all of a row kept, one token
of it, and candidates that end in every place of the last vector of 4."""
import numpy as np
import pytest

from tests.test_gpu_kv_cache import Cache, _evict, _table, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("n", [8192, 8193, 20002, 32768, 32771])
def test_shared_rows(cuda, n, ties):
    torch = _torch()
    rng = np.random.default_rng(n + ties)
    P, B = 512, 2
    width = -(-n // P)
    c = Cache(cuda, rng, "int8", 2 * B * width, P, 1)
    both = _table(rng, B, 2 * width, 2 * B * width)
    lens = [n, n - 4097]
    w = rng.integers(0, 9, size=(B, 1, n)) if ties else rng.exponential(size=(B, 1, n))
    w = torch.from_numpy(w.astype(np.float32)).to(cuda)
    for recent in (0, 1, 2, 3):
        for budget in (recent + 1, 130, n - 4100, n - 3 if recent == 2 else n - 5000):
            what = f"shared rows n={n} ties={ties} budget={budget} recent={recent}"
            print(what, flush=True)
            _evict(cuda, c, both[:, :width], both[:, width:], lens, w, budget, recent, what)
