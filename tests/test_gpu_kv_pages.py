"""Forking and compacting a paged cache on the GPU against tests/_pages_reference.py: whole
numbers and bytes, equal one by one; every byte that is not copied keeps its value."""
import random

import pytest

from tests import _pages_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = ("bf16", "e4m3", "int8")


def _cache(torch, dev, pages, P, H, dtype, seed=1, blocks=True):
    """(k, v, scales by name): random bytes and scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    t = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[dtype]
    n = 2 if dtype == "bf16" else 1
    kv = [torch.randint(0, 256, (pages, P, H, 128 * n), generator=g, device=dev, dtype=torch.uint8).view(t) for _ in range(2)]
    scales = {}
    if dtype != "bf16" and blocks:
        scales = {s: torch.rand((pages, H), generator=g, device=dev) for s in ("k_scale", "v_scale")}
    return kv[0], kv[1], scales


def _bytes(t):
    import torch
    return t.contiguous().view(-1).view(torch.uint8)


def _state(k, v, scales):
    return [t.clone() for t in (k, v, *scales.values())]


def _expect(state, copies):
    """The caches and scales after copies of (source, destination, slots or None)."""
    import torch
    out = [t.clone() for t in state]
    for src, dst, slots in copies:
        for i, (new, old) in enumerate(zip(out, state)):
            n, o = (new.view(torch.int16), old.view(torch.int16)) if new.dtype == torch.bfloat16 else (
                (new.view(torch.uint8), old.view(torch.uint8)) if new.element_size() == 1 else (new, old))
            if i < 2:
                n[dst, :slots] = o[src, :slots]
            else:
                n[dst] = o[src]
    return out


def _same(a, b):
    import torch
    return all(torch.equal(_bytes(x), _bytes(y)) for x, y in zip(a, b))


def _random_rows(r, B, W, P, num_pages, share=False):
    """A table of distinct pages (or, share, rows that begin alike), -1 and stray numbers behind them, and lengths."""
    pages = list(range(num_pages))
    r.shuffle(pages)
    table, lens = [], []
    for b in range(B):
        n = r.choice((0, 1, P - 1, P, P + 1, W * P, r.randint(0, W * P)))
        n = min(n, W * P)
        cells = [pages.pop() for _ in range(-(-n // P))]
        if share and table:
            k = min(n // P, lens[-1] // P)
            pages += cells[:k]
            cells[:k] = table[-1][:k]
        lens.append(n)
        table.append(cells + [r.choice((-1, num_pages, 7)) for _ in range(W - len(cells))])
    return table, lens


def _t(torch, dev, x, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device=dev)
    return t if shape is None else t.reshape(shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,W,P,H", [(1, 1, 1, 16, 1), (1, 8, 5, 16, 2), (4, 16, 9, 32, 4), (7, 5, 6, 64, 8), (3, 9, 40, 1, 3),
                                       (5, 33, 3, 128, 2), (20, 300, 4, 8, 1), (2, 1500, 2, 4, 1)])
@pytest.mark.parametrize("with_held", (False, True))
def test_fork(cuda, dtype, B, N, W, P, H, with_held):
    import torch
    import cuda_llm_ops_amd as fg
    for seed in range(4):
        r = random.Random(f"{B} {N} {W} {P} {seed}")
        print(dtype, B, N, W, P, H, with_held, seed, flush=True)
        num_pages = B * W + r.choice((0, 3, N * 2 + 40))
        table, lens = _random_rows(r, B, W, P, num_pages, share=seed % 2 == 1)
        parents = [r.choice((-1, B, r.randrange(B), 0)) for _ in range(N)]
        new = [r.choice((-3, 0, 1, P, r.randint(0, 3 * P))) for _ in range(N)]
        held = [r.random() < 0.3 for _ in range(num_pages)] if with_held else None
        width = r.choice((None, W, W + 2, max(1, W - 2)))
        k, v, scales = _cache(torch, cuda, num_pages, P, H, dtype, seed)
        state = _state(k, v, scales)
        want, want_lens, copies, left = ref.fork(table, lens, P, num_pages, parents, new, held, width)
        out = fg.fork_kv_paged(k, v, _t(torch, cuda, table, (B, W)), _t(torch, cuda, lens), parents=_t(torch, cuda, parents),
                               new_lens=_t(torch, cuda, new), held=None if held is None else torch.tensor(held, device=cuda),
                               max_pages=width, **scales)
        assert out[0].tolist() == want and out[1].tolist() == want_lens and out[2].tolist() == [left]
        assert _same([k, v, *scales.values()], _expect(state, copies))


def test_fork_forms(cuda):
    """No parents, no new tokens; no new rows; an empty old table; a whole-cache scale; given outputs in wider tables."""
    import torch
    import cuda_llm_ops_amd as fg
    k, v, _ = _cache(torch, cuda, 20, 16, 2, "e4m3", blocks=False)
    state = _state(k, v, {})
    table = [[3, 5, -1], [8, 5, 2]]
    t, n = _t(torch, cuda, table), _t(torch, cuda, [20, 40])
    out = fg.fork_kv_paged(k, v, t, n, k_scale=0.5, v_scale=2.0)
    assert out[0].tolist() == table and out[1].tolist() == [20, 40] and out[2].tolist() == [16]
    out = fg.fork_kv_paged(k, v, t, n, new_lens=_t(torch, cuda, [30, 9]))
    assert out[0].tolist() == ref.fork(table, [20, 40], 16, 20, None, [30, 9])[0]
    assert _same([k, v], state)
    out = fg.fork_kv_paged(k, v, t, n, parents=_t(torch, cuda, [], (0,)))
    assert out[0].shape == (0, 3) and out[2].tolist() == [20]
    out = fg.fork_kv_paged(k, v, t[:0], n[:0], parents=_t(torch, cuda, [-1, 0]), new_lens=_t(torch, cuda, [17, 0]))
    assert out[0].tolist() == [[0, 1, -1], [-1, -1, -1]] and out[1].tolist() == [0, 0] and out[2].tolist() == [18]
    out = fg.fork_kv_paged(k, v, t[:0, :0], n[:0], parents=_t(torch, cuda, [-1]), new_lens=_t(torch, cuda, [17]), max_pages=4)
    assert out[0].tolist() == [[0, 1, -1, -1]]
    wide = torch.full((4, 10), 77, dtype=torch.int32, device=cuda)
    lens, left = torch.zeros(4, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    before = wide._version
    want = ref.fork(table, [20, 40], 16, 20, [1, 1, 0, 1], [5, 5, 5, 60])
    out = fg.fork_kv_paged(k, v, t, n, parents=_t(torch, cuda, [1, 1, 0, 1]), new_lens=_t(torch, cuda, [5, 5, 5, 60]),
                           new_block_table=wide[:, 2:5], new_seqlens=lens, num_free=left)
    assert wide[:, 2:5].tolist() == want[0] and lens.tolist() == want[1] and left.tolist() == [want[3]]
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 5:] == 77).all()) and wide._version > before
    assert out[0].data_ptr() == wide[:, 2:5].data_ptr()
    assert _same([k, v], _expect(state, want[2]))


@pytest.mark.parametrize("offset", (0, 1, 3))
def test_held_of_any_value_and_address(cuda, offset):
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(offset)
    B, W, P, H, pages = 3, 30, 1, 1, 211
    table, lens = _random_rows(r, B, W, P, pages)
    marks = [r.choice((0, 0, 1, 0x7F, 0x80, 0xFF)) for _ in range(pages)]
    held = torch.tensor([9] * offset + marks, dtype=torch.uint8, device=cuda)[offset:]
    new = [5, 0, 40]
    k, v, _ = _cache(torch, cuda, pages, P, H, "bf16")
    state = _state(k, v, {})
    want, want_lens, copies, left = ref.fork(table, lens, P, pages, None, new, marks, 70)
    out = fg.fork_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens), new_lens=_t(torch, cuda, new), held=held, max_pages=70)
    assert out[0].tolist() == want and out[1].tolist() == want_lens and out[2].tolist() == [left]
    state = _expect(state, copies)
    want, moves, used = ref.compact(table, lens, P, pages, marks)
    out = fg.compact_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens), held=held)
    assert out[0].tolist() == want and out[1].tolist() == [used]
    assert _same([k, v], _expect(state, [(a, b, None) for a, b in moves]))


def test_fork_large(cuda):
    """Many pages (more words than one round of the scan), long rows, many rows, nothing free."""
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(5)
    for num_pages, B, N, W in ((200_000, 40, 64, 3000), (70_000, 3, 3000, 20), (40 * 100, 40, 60, 100)):
        P = 16
        k = torch.zeros((num_pages, P, 1, 128), dtype=torch.int8, device=cuda)
        k.view(num_pages, -1)[:, ::64] = torch.randint(-128, 128, (num_pages, 32), dtype=torch.int8, device=cuda)
        v = k.flip(0).contiguous()
        scales = {s: torch.rand((num_pages, 1), device=cuda) for s in ("k_scale", "v_scale")}
        state = _state(k, v, scales)
        pages = list(range(num_pages))
        r.shuffle(pages)
        lens = [r.randint(W * P // 2, W * P) for _ in range(B)]
        table = [[pages.pop() if j * P < n else -1 for j in range(W)] for n in lens]
        parents, new = [r.randrange(B) for _ in range(N)], [r.randint(0, 40) for _ in range(N)]
        want, want_lens, copies, left = ref.fork(table, lens, P, num_pages, parents, new)
        out = fg.fork_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens), parents=_t(torch, cuda, parents),
                               new_lens=_t(torch, cuda, new), **scales)
        assert out[0].tolist() == want and out[1].tolist() == want_lens and out[2].tolist() == [left]
        assert _same([k, v, *scales.values()], _expect(state, copies))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,W,P,H", [(1, 1, 16, 1), (4, 9, 32, 4), (7, 6, 64, 8), (3, 40, 1, 3), (40, 5, 8, 2), (2, 3, 256, 5)])
@pytest.mark.parametrize("with_held", (False, True))
def test_compact(cuda, dtype, B, W, P, H, with_held):
    import torch
    import cuda_llm_ops_amd as fg
    for seed in range(4):
        r = random.Random(f"{B} {W} {P} {seed}")
        print(dtype, B, W, P, H, with_held, seed, flush=True)
        num_pages = B * W + r.choice((0, 1, 40, 3 * B * W))
        table, lens = _random_rows(r, B, W, P, num_pages, share=seed % 2 == 1)
        held = [r.random() < 0.3 for _ in range(num_pages)] if with_held else None
        k, v, scales = _cache(torch, cuda, num_pages, P, H, dtype, seed)
        state = _state(k, v, scales)
        want, moves, used = ref.compact(table, lens, P, num_pages, held)
        out = fg.compact_kv_paged(k, v, _t(torch, cuda, table, (B, W)), _t(torch, cuda, lens),
                                  held=None if held is None else torch.tensor(held, device=cuda).to(torch.uint8) * 3, **scales)
        assert out[0].tolist() == want and out[1].tolist() == [used]
        assert _same([k, v, *scales.values()], _expect(state, [(a, b, None) for a, b in moves]))


def test_compact_forms(cuda):
    """Nothing in use; everything held; entries outside the cache; lengths below 0 and past the table; given outputs."""
    import torch
    import cuda_llm_ops_amd as fg
    k, v, scales = _cache(torch, cuda, 50, 16, 2, "int8")
    state = _state(k, v, scales)
    t = _t(torch, cuda, [[40, 41, -1], [42, 99, 49], [43, 44, 45]])
    out = fg.compact_kv_paged(k, v, t, _t(torch, cuda, [0, -5, 0]), **scales)
    assert bool((out[0] == -1).all()) and out[1].tolist() == [0]
    held = torch.ones(50, dtype=torch.bool, device=cuda)
    out = fg.compact_kv_paged(k, v, t, _t(torch, cuda, [20, 48, 1]), held=held, **scales)
    assert out[0].tolist() == [[40, 41, -1], [42, 99, 49], [43, -1, -1]] and out[1].tolist() == [50]
    assert _same([k, v, *scales.values()], state)
    out = fg.compact_kv_paged(k, v, t[:0], _t(torch, cuda, [], (0,)), **scales)
    assert out[0].shape == (0, 3) and out[1].tolist() == [0]
    new, used = torch.zeros(3, 8, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    lens = [20, 1000, 33]
    want, moves, n = ref.compact(t.tolist(), lens, 16, 50)
    fg.compact_kv_paged(k, v, t, _t(torch, cuda, lens), new_block_table=new[:, 1:4], num_used=used, **scales)
    assert new[:, 1:4].tolist() == want and used.tolist() == [n] and bool((new[:, 4:] == 0).all())
    assert _same([k, v, *scales.values()], _expect(state, [(a, b, None) for a, b in moves]))


def test_compact_large(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(6)
    num_pages, B, W, P = 300_000, 60, 2500, 16
    k = torch.randint(-128, 128, (num_pages, P, 1, 128), dtype=torch.int8, device=cuda)
    v = k.flip(0).contiguous()
    scales = {s: torch.rand((num_pages, 1), device=cuda) for s in ("k_scale", "v_scale")}
    state = _state(k, v, scales)
    pages = list(range(num_pages))
    r.shuffle(pages)
    lens = [r.randint(0, W * P) for _ in range(B)]
    table = [[pages.pop() if j * P < n else -1 for j in range(W)] for n in lens]
    want, moves, used = ref.compact(table, lens, P, num_pages)
    out = fg.compact_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens), **scales)
    assert out[0].tolist() == want and out[1].tolist() == [used]
    src, dst = (torch.tensor(x, device=cuda) for x in zip(*moves))
    for t, s in zip((k, v, *scales.values()), state):
        s[dst] = s[src]
        assert torch.equal(t, s)


@pytest.mark.parametrize("with_held", (False, True))
def test_compact_many_bytes(cuda, with_held):
    """A small table of large pages: planned in one launch and copied in another."""
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(7)
    B, W, P, H, pages = 5, 9, 4096, 8, 90
    table, lens = _random_rows(r, B, W, P, pages, share=True)
    held = [r.random() < 0.2 for _ in range(pages)] if with_held else None
    k, v, _ = _cache(torch, cuda, pages, P, H, "bf16")
    state = _state(k, v, {})
    want, moves, used = ref.compact(table, lens, P, pages, held)
    assert moves
    out = fg.compact_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens),
                              held=None if held is None else torch.tensor(held, device=cuda))
    assert out[0].tolist() == want and out[1].tolist() == [used]
    assert _same([k, v], _expect(state, [(a, b, None) for a, b in moves]))


@pytest.mark.parametrize("width", (3, 20000))
def test_offsets_past_32_bits(cuda, width):
    """Pages at both ends of a cache of more than 2^32 bytes, planned in either form."""
    import torch
    import cuda_llm_ops_amd as fg
    P, H, pages = 64, 8, 40_000
    k, v = (torch.zeros(pages, P, H, 128, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    top = pages - 6
    for i, page in enumerate((top, top + 1, top + 2)):
        k[page] = i + 1
        v[page] = -i - 1
    table, lens = [[top, top + 1] + [-1] * (width - 2), [top, top + 2] + [-1] * (width - 2)], [100, 70]
    held = torch.ones(pages, dtype=torch.bool, device=cuda)
    held[top:] = False
    want, want_lens, copies, left = ref.fork(table, lens, P, pages, [0, 0, 1], [30, 0, 0], held.tolist())
    assert [c[1] > top for c in copies] == [True]
    out = fg.fork_kv_paged(k, v, _t(torch, cuda, table), _t(torch, cuda, lens), parents=_t(torch, cuda, [0, 0, 1]),
                           new_lens=_t(torch, cuda, [30, 0, 0]), held=held)
    assert out[0].tolist() == want and out[1].tolist() == want_lens and out[2].tolist() == [left]
    src, dst, slots = copies[0]
    assert bool((k[dst, :slots] == k[src, :slots]).all()) and bool((v[dst, :slots] == -2).all())
    assert not bool(k[dst, slots:].any())
    moved, moves, used = ref.compact(want, want_lens, P, pages)
    was = {s: (k[s].clone(), v[s].clone()) for s, _ in moves}
    out = fg.compact_kv_paged(k, v, out[0], out[1])
    assert out[0].tolist() == moved and out[1].tolist() == [used] == [len(moves)]
    for s, d in moves:
        assert torch.equal(k[d], was[s][0]) and torch.equal(v[d], was[s][1])


def test_strided_caches(cuda):
    """K and V interleaved in one tensor, heads before slots, scales by columns."""
    import torch
    import cuda_llm_ops_amd as fg
    both = torch.randint(-128, 128, (30, 2, 4, 16, 128), dtype=torch.int8, device=cuda)
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    sc = torch.rand((4, 2, 30), device=cuda)
    scales = dict(k_scale=sc[:, 0].t(), v_scale=sc[:, 1].t())
    state = [t.clone(memory_format=torch.contiguous_format) for t in (k, v, *scales.values())]
    table, lens = [[29, 3, 17], [11, 28, -1]], [45, 30]
    want, want_lens, copies, left = ref.fork(table, lens, 16, 30, [0, 1, 1, 0], [4, 4, 40, 4])
    t, n = _t(torch, cuda, table), _t(torch, cuda, lens)
    out = fg.fork_kv_paged(k, v, t, n, parents=_t(torch, cuda, [0, 1, 1, 0]), new_lens=_t(torch, cuda, [4, 4, 40, 4]), **scales)
    assert out[0].tolist() == want and out[2].tolist() == [left]
    state = _expect(state, copies)
    assert _same([k, v, *scales.values()], state)
    want, moves, _ = ref.compact(want, want_lens, 16, 30)
    out = fg.compact_kv_paged(k, v, out[0], out[1], **scales)
    assert out[0].tolist() == want
    assert _same([k, v, *scales.values()], _expect(state, [(a, b, None) for a, b in moves]))


def test_another_stream_and_graphs(cuda):
    """On a stream of its own, and in two captured graphs whose replays follow changed tables."""
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(3)
    B, N, W, P, num_pages = 6, 12, 7, 16, 120
    k, v, scales = _cache(torch, cuda, num_pages, P, 2, "int8")
    table, lens = _random_rows(r, B, W, P, num_pages)
    t, n = _t(torch, cuda, table), _t(torch, cuda, lens)
    parents, new = _t(torch, cuda, [r.randrange(B) for _ in range(N)]), _t(torch, cuda, [r.randint(0, 20) for _ in range(N)])

    def step():
        a = fg.fork_kv_paged(k, v, t, n, parents=parents, new_lens=new, **scales)
        return a + fg.compact_kv_paged(k, v, a[0], a[1], **scales)

    def expected():
        want, want_lens, copies, left = ref.fork(t.tolist(), n.tolist(), P, num_pages, parents.tolist(), new.tolist())
        state = _expect(_state(k, v, scales), copies)
        to, moves, used = ref.compact(want, want_lens, P, num_pages)
        return [want, want_lens, [left], to, [used]], _expect(state, [(a, b, None) for a, b in moves])

    want, state = expected()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert [x.tolist() for x in got] == want and _same([k, v, *scales.values()], state)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for i in range(4):
        table, lens = _random_rows(r, B, W, P, num_pages, share=i % 2 == 0)
        t.copy_(_t(torch, cuda, table))
        n.copy_(_t(torch, cuda, lens))
        parents.copy_(_t(torch, cuda, [r.randrange(-1, B) for _ in range(N)]))
        for graph, got in graphs:
            want, state = expected()
            graph.replay()
            torch.cuda.synchronize()
            assert [x.tolist() for x in got] == want and _same([k, v, *scales.values()], state), i


def test_fork_then_append(cuda):
    """Beams go on from their best for some steps: each keeps exactly the tokens of its own history."""
    import torch
    import cuda_llm_ops_amd as fg
    r = random.Random(9)
    P, H, N, W, num_pages = 16, 2, 6, 8, 60
    k = torch.zeros((num_pages, P, H, 128), dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    table = torch.full((1, W), -1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda)
    history = [[]]
    stamp = 0
    for step in range(14):
        parents = [r.randrange(len(history)) for _ in range(N)]
        new = [r.choice((1, 1, 2, 11)) for _ in range(N)]
        history = [list(history[p]) for p in parents]
        table, lens, left = fg.fork_kv_paged(k, v, table, lens, parents=_t(torch, cuda, parents),
                                             new_lens=_t(torch, cuda, new))
        assert int(left) >= 0
        x = torch.zeros((N, max(new), H, 128), dtype=torch.bfloat16, device=cuda)
        for i, m in enumerate(new):
            for j in range(m):
                stamp = stamp % 250 + 1
                x[i, j] = stamp
                history[i].append(stamp)
        if max(len(h) for h in history) > W * P:
            break
        fg.append_kv_paged(x, -x, k, v, table, lens, new_lens=_t(torch, cuda, new))
        lens = lens + _t(torch, cuda, new)
        if step % 4 == 3:
            table, _ = fg.compact_kv_paged(k, v, table, lens)
        for i, h in enumerate(history):
            pages = table[i, :-(-len(h) // P)].long()
            assert k[pages].reshape(-1, H, 128)[:len(h), 1, 77].tolist() == h, (step, i)
            assert v[pages].reshape(-1, H, 128)[:len(h), 0, 3].tolist() == [-a for a in h], (step, i)


def _page_structs():
    import ctypes as C
    two, three = C.c_int64 * 2, C.c_int64 * 3

    class Cache(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_scales", "v_scales")] + [
            (n, C.c_int32) for n in ("kv_dtype", "num_kv_heads", "head_dim", "page_size", "num_pages")] + [
            ("k_scale", C.c_float), ("v_scale", C.c_float), ("k_stride", three), ("v_stride", three),
            ("k_scales_stride", two), ("v_scales_stride", two)]

    class Fork(C.Structure):
        _fields_ = [("cache", Cache)] + [(n, C.c_void_p) for n in (
            "block_table", "seqlens", "parents", "new_lens", "held", "new_block_table", "new_seqlens", "num_free")] + [
            ("block_table_stride", C.c_int64), ("new_block_table_stride", C.c_int64)] + [
            (n, C.c_int32) for n in ("batch", "max_pages", "new_batch", "new_max_pages")] + [
            ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]

    class Compact(C.Structure):
        _fields_ = [("cache", Cache)] + [(n, C.c_void_p) for n in (
            "block_table", "seqlens", "held", "new_block_table", "num_used")] + [
            ("block_table_stride", C.c_int64), ("new_block_table_stride", C.c_int64)] + [
            (n, C.c_int32) for n in ("batch", "max_pages")] + [("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]

    return Cache, Fork, Compact


CacheArgs, ForkArgs, CompactArgs = _page_structs()


@pytest.mark.parametrize("width", (9, 9000))
def test_workspaces_of_the_c_abi(cuda, width):
    """A narrow table needs no workspace; of a wide one (planned in launches of its own) too small and
    misaligned ones are refused, and one that is large enough gives what the library's gives."""
    import ctypes
    import torch
    import cuda_llm_ops_amd as fg
    L = ctypes.CDLL(fg.LIB_PATH)
    r = random.Random(width)
    B, N, W, P, H, pages = 4, 6, 9, 16, 2, 60
    table, lens = _random_rows(r, B, W, P, pages)
    table = [row + [5] * (width - W) for row in table]
    parents, new = [3, 0, 0, -1, 2, 0], [4, 0, 40, 17, 1, 3]
    stream = torch.cuda.current_stream().cuda_stream
    for kind in ("fork", "compact"):
        k, v, _ = _cache(torch, cuda, pages, P, H, "bf16")
        state = _state(k, v, {})
        t, ln, pa, nw = (_t(torch, cuda, x) for x in (table, lens, parents, new))
        a = ForkArgs() if kind == "fork" else CompactArgs()
        a.cache.kv_dtype, a.cache.num_kv_heads, a.cache.head_dim, a.cache.page_size, a.cache.num_pages = 0, H, 128, P, pages
        a.cache.k, a.cache.v, a.cache.k_scale, a.cache.v_scale = k.data_ptr(), v.data_ptr(), 1.0, 1.0
        a.cache.k_stride[:], a.cache.v_stride[:] = [P * H * 128, H * 128, 128], [P * H * 128, H * 128, 128]
        a.block_table, a.seqlens, a.block_table_stride, a.batch, a.max_pages = t.data_ptr(), ln.data_ptr(), width, B, width
        rows = N if kind == "fork" else B
        out, out_lens, count = (torch.empty(n, dtype=torch.int32, device=cuda) for n in ((rows, width), (rows,), (1,)))
        a.new_block_table, a.new_block_table_stride = out.data_ptr(), width
        if kind == "fork":
            a.parents, a.new_lens, a.new_seqlens, a.num_free = pa.data_ptr(), nw.data_ptr(), out_lens.data_ptr(), count.data_ptr()
            a.new_batch, a.new_max_pages = N, width
            want, want_lens, copies, want_count = ref.fork(table, lens, P, pages, parents, new)
        else:
            a.num_used = count.data_ptr()
            want, moves, want_count = ref.compact(table, lens, P, pages)
            copies = [(s, d, None) for s, d in moves]
        fn = getattr(L, f"fgqa_kv_{kind}")
        fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
        need = ctypes.c_size_t(1 << 40)
        assert getattr(L, f"fgqa_kv_{kind}_workspace_bytes")(ctypes.byref(a), ctypes.byref(need)) == 0
        assert (need.value > 0) == (width > 9) and need.value < 1 << 20
        work = torch.empty(need.value + 256, dtype=torch.uint8, device=cuda)
        if need.value > 0:
            for ws, n, status in ((work.data_ptr(), need.value - 1, -3), (work.data_ptr() + 4, need.value, -2), (None, need.value, -3)):
                a.workspace, a.workspace_bytes = ws, n
                assert fn(ctypes.byref(a), stream) == status
        for ws, n in ((work.data_ptr(), need.value), (None, 0)):
            for x, s in zip((k, v), state):
                x.copy_(s)
            for x in (out, out_lens, count):
                x.fill_(-77)
            a.workspace, a.workspace_bytes = ws, n
            assert fn(ctypes.byref(a), stream) == 0
            assert out.tolist() == want and count.tolist() == [want_count]
            assert kind == "compact" or out_lens.tolist() == want_lens
            assert _same([k, v], _expect(state, copies))


@pytest.mark.parametrize("width", (9, 9000))
def test_no_new_rows_of_the_c_abi(cuda, width):
    """Every sequence is dropped: the old rows are not read (here there are none), the pages are counted."""
    import ctypes
    import torch
    import cuda_llm_ops_amd as fg
    P, H, pages = 16, 2, 60
    k, v, _ = _cache(torch, cuda, pages, P, H, "bf16")
    a = ForkArgs()
    a.cache.kv_dtype, a.cache.num_kv_heads, a.cache.head_dim, a.cache.page_size, a.cache.num_pages = 0, H, 128, P, pages
    a.cache.k, a.cache.v, a.cache.k_scale, a.cache.v_scale = k.data_ptr(), v.data_ptr(), 1.0, 1.0
    a.cache.k_stride[:], a.cache.v_stride[:] = [P * H * 128, H * 128, 128], [P * H * 128, H * 128, 128]
    held = torch.tensor([1] * 7 + [0] * (pages - 7), dtype=torch.uint8, device=cuda)
    count = torch.full((1,), -77, dtype=torch.int32, device=cuda)
    a.held, a.num_free = held.data_ptr(), count.data_ptr()
    a.block_table_stride, a.new_block_table_stride, a.batch, a.max_pages, a.new_max_pages = width, width, 4, width, width
    fn = ctypes.CDLL(fg.LIB_PATH).fgqa_kv_fork
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert fn(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert count.tolist() == [pages - 7]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_held", (False, True))
def test_wide_tables(cuda, dtype, with_held):
    """Rows that could be long: the same calls planned in launches of their own."""
    import torch
    import cuda_llm_ops_amd as fg
    for seed, (B, N, W, P, H, width) in enumerate(((4, 16, 9, 32, 4, 9000), (40, 50, 5, 8, 2, 1000), (1, 3, 6, 64, 8, 40000))):
        r = random.Random(f"{dtype} {with_held} {seed}")
        num_pages = 2 * B * W + 40
        table, lens = _random_rows(r, B, W, P, num_pages)
        parents = [r.choice((-1, B, r.randrange(B), 0)) for _ in range(N)]
        new = [r.choice((-3, 0, 1, P, r.randint(0, 3 * P))) for _ in range(N)]
        held = [r.random() < 0.3 for _ in range(num_pages)] if with_held else None
        held_t = None if held is None else torch.tensor(held, device=cuda)
        wide = [row + [-1] * (width - W) for row in table]
        k, v, scales = _cache(torch, cuda, num_pages, P, H, dtype, seed)
        state = _state(k, v, scales)
        want, want_lens, copies, left = ref.fork(wide, lens, P, num_pages, parents, new, held)
        out = fg.fork_kv_paged(k, v, _t(torch, cuda, wide), _t(torch, cuda, lens), parents=_t(torch, cuda, parents),
                               new_lens=_t(torch, cuda, new), held=held_t, **scales)
        assert out[0].tolist() == want and out[1].tolist() == want_lens and out[2].tolist() == [left]
        state = _expect(state, copies)
        assert _same([k, v, *scales.values()], state)
        want, moves, used = ref.compact(wide, lens, P, num_pages, held)
        out = fg.compact_kv_paged(k, v, _t(torch, cuda, wide), _t(torch, cuda, lens), held=held_t, **scales)
        assert out[0].tolist() == want and out[1].tolist() == [used]
        assert _same([k, v, *scales.values()], _expect(state, [(s, d, None) for s, d in moves]))
