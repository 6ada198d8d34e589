"""Eviction where the rows of weights are shorter than the sequences: the newest
tokens, which have no weight, are kept as the recent ones are."""
import numpy as np
import pytest

from tests import _kv_reference as ref
from tests.test_gpu_kv_cache import KINDS, Cache, _i32, _table, _torch

pytestmark = pytest.mark.gpu


def _run(cuda, c, table, new_table, lens, w, budget, recent, most):
    """The call, and the same from the definition: tokens at or past the row's width
    count as recent ones, and sequences are cut to `most` tokens."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    B, H, W = w.shape
    P, total = c.t[0].shape[1], table.shape[1] * c.t[0].shape[1]
    nl, nw, kept = fg.evict_kv_paged(c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens), w.to(cuda), _i32(cuda, new_table),
                                     budget=budget, recent=recent, **c.scales)
    torch.cuda.synchronize()
    assert nw.shape == w.shape and kept.shape == (B, H, budget)
    wide = np.zeros((B, H, max(total, W)), np.float32)
    wide[:, :, :W] = w.numpy()
    for b, n in enumerate(lens):
        cut, n = min(budget, most), min(n, total)
        rl, rw, rk = ref.evict(c.n[0], c.sn[0], c.n[1], c.sn[1], c.dtype, table[b:b + 1], new_table[b:b + 1], np.array([n]),
                               np.where(np.arange(wide.shape[2]) < W, wide[b:b + 1], 0), cut, max(recent, n - W))
        assert int(nl[b]) == rl[0], f"sequence {b}: length"
        assert np.array_equal(kept[b, :, :cut].cpu().numpy(), rk[0]) and bool((kept[b, :, cut:] == -1).all()), f"sequence {b}: kept"
        assert np.array_equal(nw[b].cpu().numpy(), rw[0, :, :W]), f"sequence {b}: weights"
    c.check("short weights")


@pytest.mark.parametrize("dtype,scales", KINDS)
@pytest.mark.parametrize("P", [4, 16, 128])
@pytest.mark.parametrize("budget,recent", [(100, 16), (100, 0), (400, 16), (1, 0), (250, 250)])
def test_newest_tokens_stay(cuda, budget, recent, P, dtype, scales):
    torch = _torch()
    print(f"short weights P={P} {dtype} {scales} budget={budget} recent={recent}", flush=True)
    rng = np.random.default_rng(3000 + P)
    lens, W = [640, 300, 40, 301, 500, 0], 300
    width, nwidth = -(-640 // P), -(-min(budget, 640) // P)
    pages = len(lens) * (width + nwidth)
    c = Cache(cuda, rng, dtype, pages, P, 2, scales=scales)
    both = _table(rng, len(lens), width + nwidth, pages)
    w = torch.from_numpy(rng.exponential(size=(len(lens), 2, W)).astype(np.float32))
    _run(cuda, c, both[:, :width], both[:, width:], lens, w, budget, recent, 10 ** 9)


def test_new_pages_for_the_weights_only(cuda):
    """A new block table that has pages for the weights' row but not for the budget:
    longer sequences are cut to what it holds, from the oldest and lightest on."""
    torch = _torch()
    rng = np.random.default_rng(3100)
    lens, W, P = [640, 300, 200], 300, 16
    c = Cache(cuda, rng, "int8", 3 * 60, P, 1)
    both = _table(rng, 3, 40 + 19, 3 * 60)
    w = torch.from_numpy(rng.exponential(size=(3, 1, W)).astype(np.float32))
    _run(cuda, c, both[:, :40], both[:, 40:], lens, w, 500, 20, 19 * P)


def test_lengths_past_the_table(cuda):
    """Lengths past the block table count as its tokens."""
    torch = _torch()
    rng = np.random.default_rng(3200)
    c = Cache(cuda, rng, "e4m3", 60, 16, 2)
    both = _table(rng, 2, 24, 60)
    w = torch.from_numpy(rng.exponential(size=(2, 2, 100)).astype(np.float32))
    _run(cuda, c, both[:, :20], both[:, 20:], [100000, 2 ** 31 - 1], w, 60, 9, 10 ** 9)


def test_long_rows_shared_by_workgroups(cuda):
    torch = _torch()
    rng = np.random.default_rng(3300)
    for W in (9001, 40000):
        P, n = 512, W + 700
        width = -(-n // P)
        c = Cache(cuda, rng, "int8", width + 6, P, 1)
        both = _table(rng, 1, width + 6, width + 6)
        w = torch.from_numpy(rng.exponential(size=(1, 1, W)).astype(np.float32))
        _run(cuda, c, both[:, :width], both[:, width:], [n], w, 3000, 10, 10 ** 9)


def test_weights_of_no_tokens(cuda):
    """All tokens are recent then; without new pages none is kept."""
    import cuda_llm_ops_amd as fg
    torch = _torch()
    rng = np.random.default_rng(3400)
    c = Cache(cuda, rng, "int8", 60, 16, 2)
    both = _table(rng, 2, 24, 60)
    w = torch.zeros((2, 2, 0))
    _run(cuda, c, both[:, :20], both[:, 20:], [300, 7], w, 60, 3, 10 ** 9)
    nl, nw, kept = fg.evict_kv_paged(c.t[0], c.t[1], _i32(cuda, both[:, :20]), _i32(cuda, [300, 7]), w.to(cuda),
                                     _i32(cuda, both)[:, :0], budget=60, recent=3, **c.scales)
    torch.cuda.synchronize()
    assert nl.tolist() == [0, 0] and nw.shape == (2, 2, 0) and bool((kept == -1).all())
    c.check("no new pages")
