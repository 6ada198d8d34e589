"""The decode of sequences that begin alike on the GPU against float64.

Bounds of an output element, with p the exact weights of a row (they sum to 1): P is rounded
to bf16 over shared tokens and, of bf16 and whole-cache e4m3 caches, over a sequence's own (2^-8 of
each weight), the scores' fp32 error e_s (128 products and their sum, q.k and the
exponent's rounding: (2^-18 + 2^-20 |score|) times the sum of |q k| / |q.k|, here
taken as 2^-17 sum |q k| scale) moves each weight by e_s, the output rounds to bf16 once
(2^-8 of it), and fp32 sums add 2^-17 of sum p |v|.  The LSE moves by e_s and fp32 sums."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D = 128


class Case:
    """Sequences on pages of a cache, groups of which share their first pages; everything else is filled
    with NaN (bf16, e4m3) or the largest codes."""

    def __init__(self, torch, dev, dtype, Hq, Hkv, P, shared, groups, alone=(), seed=1, scales="blocks", sigma=1.0, extra=3,
                 wide=True):
        """shared: tokens of each group; groups: each group's sequences' own tokens; alone: of those without;
        wide: rows that could be long, which small calls over block scales are not decoded one by one with."""
        r = random.Random(seed)
        self.torch, self.dev, self.dtype, self.P, self.Hq, self.Hkv = torch, dev, dtype, P, Hq, Hkv
        self.starts, self.shared = [0], list(shared)
        rows, lens = [], []
        need = sum(s // P for s in shared) + sum(-(-(s % P + n) // P) for s, g in zip(shared, groups) for n in g)
        need += sum(-(-n // P) for n in alone) + 2
        pages = list(range(need))
        r.shuffle(pages)
        for s, g in zip(shared, groups):
            first = [pages.pop() for _ in range(s // P)]
            for n in g:
                rows.append(first + [pages.pop() for _ in range(-(-(s % P + n) // P))])
                lens.append(s + n)
            self.starts.append(len(rows))
        for n in alone:
            rows.append([pages.pop() for _ in range(-(-n // P))])
            lens.append(n)
        self.lens = lens
        W = max([len(x) for x in rows] + [1]) + extra
        if wide and dtype != "bf16" and scales == "blocks" and rows:
            W = max(W, 1152 * 256 // (len(rows) * Hkv * P) + 1)
        # (entries behind a sequence's pages are nobody's)
        self.table = torch.tensor([x + [r.choice((-1, need + 5, 0))] * (W - len(x)) for x in rows], dtype=torch.int32,
                                  device=dev).reshape(len(rows), W)
        g = torch.Generator(device="cpu").manual_seed(seed)
        t = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[dtype]
        self.kw = {}
        self.cache, self.values = [], []
        used = torch.zeros(need, P, dtype=torch.bool)
        for row, n in zip(rows, lens):
            for j, page in enumerate(row):
                used[page, :max(0, min(P, n - j * P))] = True
        for name in ("k", "v"):
            x = sigma * torch.randn(need, P, Hkv, D, generator=g)
            x *= 0.5 + torch.rand(1, 1, Hkv, 1, generator=g)
            if dtype == "bf16":
                c, v = x.to(t), x.to(t).double()
                c = torch.where(used[:, :, None, None], c, torch.tensor(float("nan"), dtype=t))
            else:
                q = 448.0 if dtype == "e4m3" else 127.0
                s = torch.full((need, Hkv), 0.03125) if scales == "whole" else torch.exp2(
                    torch.ceil(torch.log2(x.abs().amax(dim=(1, 3)) / q)))
                y = (x / s[:, None, :, None]).clamp(-q, q)
                c = y.to(t) if dtype == "e4m3" else y.round().to(t)
                v = c.double() * s.double()[:, None, :, None]
                bad = torch.tensor(0x7F, dtype=torch.uint8)   # e4m3's NaN, int8's 127
                c = torch.where(used[:, :, None, None], c.view(torch.uint8), bad).view(t)
                self.kw[name + "_scale"] = 0.03125 if scales == "whole" else s.to(dev)
            self.cache.append(c.to(dev))
            self.values.append(v.numpy())
        self.q = torch.randn(len(rows), Hq, D, generator=g).to(torch.bfloat16).to(dev)
        self.n = torch.tensor(lens, dtype=torch.int32, device=dev)

    def ints(self, x):
        return self.torch.tensor(x, dtype=self.torch.int32, device=self.dev)

    def run(self, starts=None, shared=None, **kw):
        import cuda_llm_ops_amd as fg
        torch = self.torch
        lse = torch.full((len(self.lens), self.Hq), float("nan"), device=self.dev)
        out = fg.decode_flash_gqa_paged_shared(
            self.q, *self.cache, self.table, self.n, self.ints(self.starts if starts is None else starts),
            self.ints(self.shared if shared is None else shared), lse=lse, **{**self.kw, **kw})
        return out, lse

    def check(self, out, lse, scale=None, lens=None):
        scale = 1 / math.sqrt(D) if scale is None else scale
        q, table = self.q.double().cpu().numpy(), self.table.cpu().numpy()
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        G = self.Hq // self.Hkv
        for b, n in enumerate(self.lens if lens is None else lens):
            if n <= 0:
                assert (out[b] == 0).all() and (lse[b] == -np.inf).all(), b
                continue
            pages = table[b, :-(-n // self.P)]
            k, v = (x[pages].reshape(-1, self.Hkv, D)[:n] for x in self.values)
            for h in range(self.Hkv):
                rows = slice(h * G, (h + 1) * G)
                s = scale * (q[b, rows] @ k[:, h].T)
                e = 2.0 ** -17 * abs(scale) * (np.abs(q[b, rows]) @ np.abs(k[:, h]).T)
                m = s.max(axis=1, keepdims=True)
                p = np.exp(s - m)
                total = p.sum(axis=1, keepdims=True)
                p /= total
                want = p @ v[:, h]
                moved = (p * (2.0 ** -8 + 2.0 ** -17 + e + (p * e).sum(axis=1, keepdims=True))) @ np.abs(v[:, h])
                bound = 2.0 ** -8 * np.abs(want) + 1.01 * moved
                d = np.abs(out[b, rows] - want)
                assert np.isfinite(d).all() and (d <= bound).all(), (b, h, float((d - bound).max()), float(d.max()))
                want = (m + np.log(total))[:, 0]
                d = np.abs(lse[b, rows] - want)
                assert (d <= (p * e).sum(axis=1) + 2.0 ** -17 + 2.0 ** -22 * np.abs(want)).all(), (b, h, float(d.max()))


@pytest.mark.parametrize("dtype,scales", [("bf16", None), ("e4m3", "blocks"), ("e4m3", "whole"), ("int8", "blocks")])
@pytest.mark.parametrize("Hq,Hkv,P,shared,groups,alone", [
    (4, 1, 16, [256], [[5, 1]], []),
    (16, 2, 16, [400], [[3, 50, 1, 130, 0, 17, 64, 9]], []),
    (8, 8, 64, [1000, 700], [[1, 2, 3], [40] * 5], [33, 1, 600]),
    (28, 4, 32, [130, 2000], [[10] * 21, [600, 7]], [5]),
    (16, 1, 128, [3000], [[20, 300, 1]], [2000]),
    (32, 2, 8, [333], [[1] * 17], []),
    (6, 3, 4, [200, 150], [[4, 5], [6, 130]], [7]),
    (5, 5, 1, [137], [[4, 1, 30, 2]], []),
    (64, 8, 16, [512], [[1] * 33], []),
    (12, 4, 256, [700], [[1, 300, 250]], []),
])
def test_against_float64(cuda, dtype, scales, Hq, Hkv, P, shared, groups, alone):
    import torch
    print(dtype, scales, Hq, Hkv, P, shared, [len(g) for g in groups], alone, flush=True)
    c = Case(torch, cuda, dtype, Hq, Hkv, P, shared, groups, alone, scales=scales)
    out, lse = c.run()
    c.check(out, lse)
    again, lse2 = c.run()
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", ("e4m3", "int8"))
def test_small_calls(cuda, dtype):
    """Block scales and few tokens: each sequence on its own, as decode_flash_gqa_paged has it."""
    import torch
    import cuda_llm_ops_amd as fg
    for Hq, Hkv, P, shared, groups, alone in ((16, 2, 16, [400], [[3, 50, 1, 130, 0, 17, 64, 9]], []), (8, 8, 64, [300], [[1, 2]], [33]),
                                              (4, 1, 8, [137], [[40] * 5], []), (6, 3, 1, [0], [[1]], [7])):
        c = Case(torch, cuda, dtype, Hq, Hkv, P, shared, groups, alone, wide=False)
        out, lse = c.run()
        c.check(out, lse)
        want_lse = torch.empty_like(lse)
        want = fg.decode_flash_gqa_paged(c.q, *c.cache, c.table, c.n, lse=want_lse, **c.kw)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        work = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
        again, lse2 = c.run(workspace=work)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
        c.n[0] = 0
        c.check(*c.run(), lens=[0] + c.lens[1:])


@pytest.mark.parametrize("dtype", ("bf16", "int8"))
def test_no_sharing_at_all(cuda, dtype):
    """No groups; groups of one sequence; shared lengths of 0 or below; less than a page."""
    import torch
    c = Case(torch, cuda, dtype, 16, 2, 64, [300, 200], [[40, 7, 700], [1, 2]], [90, 5000])
    for starts, shared in (([0], []), ([0, 1, 2], [300, 300]), ([0, 3, 5], [0, -7]), ([0, 3, 5], [63, 50]), ([7, 7], [100])):
        c.check(*c.run(starts, shared))


@pytest.mark.parametrize("dtype", ("bf16", "e4m3"))
def test_odd_groups(cuda, dtype):
    """Starts that are not ascending or outside the batch, more groups than sequences, shared lengths past the
    sequences', part of what is shared, sequences without tokens in a group."""
    import torch
    c = Case(torch, cuda, dtype, 8, 2, 16, [512], [[40, 7, 300, 1, 20, 2]], [90])
    for starts, shared in (([0, 6], [512]), ([-5, 6], [300]), ([0, 6], [1 << 30]), ([2, 5], [511]), ([0, 3, 3, 6], [512, 100, 256]),
                           ([0, 4, 2, 6], [512, 512, 512]), ([3, 1, 6, 99], [512, 512, 90]), ([0, 2, 4, 6] + [6] * 30, [512] * 33)):
        if shared == [1 << 30]:   # (then all sequences of the group do share what the shortest has)
            same = c.table.clone()
            c.check(*c.run(starts, [512]))
            assert torch.equal(same, c.table)
            continue
        print(starts, shared, flush=True)
        c.check(*c.run(starts, shared))
    lens = list(c.lens)
    for change in ({1: 0}, {0: 0, 3: -4}, {0: 0, 1: 0, 2: 0, 3: 0, 4: 0}, {i: 0 for i in range(7)}, {2: 100}, {4: 3}):
        now = [change.get(i, n) for i, n in enumerate(lens)]
        c.n.copy_(c.ints(now))
        c.check(*c.run(), lens=now)
    c.n.copy_(c.ints(lens))
    # a row of the table whose sequence is empty is not read: the next one's is
    c.n[0] = 0
    c.table[0] = 1 << 20
    now = [0] + lens[1:]
    c.check(*c.run(), lens=now)


def test_many_groups(cuda):
    import torch
    c = Case(torch, cuda, "int8", 4, 2, 16, [128 + 16 * (i % 3) for i in range(1100)], [[3, 20]] * 1100)
    c.check(*c.run())


def test_odd_groups_of_many(cuda):
    """As test_odd_groups, of more sequences or groups than the decode's workgroups plan for themselves."""
    import torch
    c = Case(torch, cuda, "int8", 4, 2, 16, [256], [[1 + i % 5 for i in range(300)]], [40, 300])
    for starts, n in (([0, 300], 1), ([-5, 300], 1), ([0, 200, 100, 300], 3), ([299, 1, 300, 9999], 3),
                      (list(range(0, 302, 2)) + [300] * 250, 400)):
        print(starts[:4], n, flush=True)
        c.check(*c.run(starts, [256] * n))
    now = [0 if i % 3 == 0 else 3 if i == 7 else n for i, n in enumerate(c.lens)]
    c.n.copy_(c.ints(now))
    c.check(*c.run(), lens=now)
    c = Case(torch, cuda, "int8", 4, 2, 16, [256], [[1 + i % 5 for i in range(30)]], [40])
    c.check(*c.run([0, 20, 10, 30] + [30] * 297, [256] * 300))


def test_long_and_large(cuda):
    """A long document: many cuts of the shared tokens; a large group: many row tiles."""
    import torch
    c = Case(torch, cuda, "bf16", 4, 1, 64, [40_000], [[1, 60, 500]])
    c.check(*c.run())
    c = Case(torch, cuda, "e4m3", 16, 1, 16, [700], [[1 + i % 9 for i in range(150)]])
    c.check(*c.run())


def test_scales_of_the_scores(cuda):
    import torch
    c = Case(torch, cuda, "int8", 8, 2, 16, [400], [[9, 200, 1]], [77])
    for scale in (0.5, -0.2, 0.0, 1e-6):
        c.check(*c.run(scale=scale), scale=scale)
    c = Case(torch, cuda, "bf16", 8, 2, 16, [400], [[9, 200, 1]], [77], sigma=6.0)
    for scale in (1.0, -0.7):
        c.check(*c.run(scale=scale), scale=scale)


def test_max_seqlen_and_given_tensors(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = Case(torch, cuda, "int8", 8, 2, 16, [400], [[9, 200, 1]], [77])
    want, want_lse = c.run()
    wide = torch.full((4, 8, 256), 3.0, dtype=torch.bfloat16, device=cuda)
    before = wide._version
    out, lse = c.run(out=wide[:, :, 64:192])
    assert torch.equal(wide[:, :, 64:192], want) and bool((wide[:, :, :64] == 3).all()) and wide._version > before
    assert out.data_ptr() == wide[:, :, 64:].data_ptr()
    out, lse = c.run(max_seqlen=405)
    c.check(out, lse, lens=[min(n, 405) for n in c.lens])
    out, lse = c.run(max_seqlen=0)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    # workspaces: too small and misaligned ones
    work = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    out, lse = c.run(workspace=work)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    with pytest.raises(fg.FgqaError, match="workspace too small"):
        c.run(workspace=work[:4096])
    with pytest.raises(fg.FgqaError, match="alignment"):
        c.run(workspace=work[16:])
    # strided queries, and ones that are copied
    q = torch.zeros(4, 8, 200, dtype=torch.bfloat16, device=cuda)
    for part in (q[:, :, 8:136], q[:, :, 3:131]):
        part.copy_(c.q)
        c.q = part
        assert torch.equal(c.run()[0], want)


def test_infinite_and_nan_values(cuda):
    """Infinite keys give weights of 0 or NaN rows, NaN values their column, in the rows that see them only."""
    import torch
    c = Case(torch, cuda, "bf16", 4, 2, 16, [256], [[40, 7, 300]], [90])
    clean, _ = c.run()
    k, v = c.cache
    page = int(c.table[1, 16])            # sequence 1's own first page
    v[page, 2, 1, 5] = float("nan")
    out, _ = c.run()
    bad = out.isnan()
    assert bool(bad[1, 2:, 5].all()) and int(bad.sum()) == 2 and torch.equal(out[~bad], clean[~bad])
    v[page, 2, 1, 5] = 0.0
    # keys whose scores are -inf for a positive query: all of a shared tile and more, then numbers
    c.q[:] = c.q.abs()
    pages = c.table[0, :10].long()
    saved = k[pages].clone()
    k[pages, :, 0, 0] = -float("inf")
    out, lse = c.run()
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
    c.values[0][pages.cpu().numpy(), :, 0, :] = 0
    # (against the same sequences without those tokens)
    q, table = c.q.double().cpu().numpy(), c.table.cpu().numpy()
    for b in range(3):
        n = c.lens[b]
        kk, vv = (x[table[b, :-(-n // 16)]].reshape(-1, 2, D)[160:n, 0] for x in c.values)
        s = q[b, :2] @ kk.T / math.sqrt(D)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        want = p @ vv / p.sum(axis=1, keepdims=True)
        d = np.abs(out[b, :2].double().cpu().numpy() - want)
        assert (d <= 2.0 ** -8 * np.abs(want) + 2.0 ** -7 * (p @ np.abs(vv)) / p.sum(axis=1, keepdims=True)).all()
    k[pages] = saved
    # own tokens of a sequence all at -inf, the shared ones numbers
    own = c.table[1, 16:17].long()
    k[own, :, 0, 0] = -float("inf")
    out, lse = c.run()
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
    # and no number at all: NaN, as 0 / 0
    k[c.table[3, :6].long(), :, 1, 0] = -float("inf")
    out, _ = c.run()
    assert bool(out[3, 2:].isnan().all()) and bool(out[:3].isfinite().all()) and bool(out[3, :2].isfinite().all())


def test_offsets_past_32_bits(cuda):
    """Pages whose bytes lie past 2^32 from the cache's start, of K and of V."""
    import torch
    c = Case(torch, cuda, "int8", 8, 8, 64, [640], [[9, 200, 1]], [77])
    far = 70_000                          # of 64 KiB each: 4.6 GB
    n = c.cache[0].shape[0]
    moved = []
    for t in c.cache:
        big = torch.zeros(far + n, 64, 8, 128, dtype=torch.int8, device=cuda)
        big[far:] = t
        moved.append(big)
    want, lse = c.run()
    c.cache = moved
    c.table += torch.where((c.table >= 0) & (c.table < n), far, 0)
    for s in ("k_scale", "v_scale"):
        c.kw[s] = torch.cat((torch.ones(far, 8, device=cuda), c.kw[s]))
    out, lse2 = c.run()
    assert torch.equal(out, want) and torch.equal(lse, lse2)


def test_another_stream_and_graphs(cuda):
    """On two streams at once, and in two captured graphs replayed after changed lengths and groups."""
    import torch
    c = Case(torch, cuda, "e4m3", 16, 2, 16, [400, 256], [[30] * 6, [100, 7, 70]], [77, 900])
    want, want_lse = c.run()
    starts, shared = c.ints(c.starts), c.ints(c.shared)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(c.run())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) and torch.equal(x, want_lse) for o, x in got)
    import cuda_llm_ops_amd as fg
    lse = torch.zeros(len(c.lens), 16, device=cuda)

    def step(lse):
        return fg.decode_flash_gqa_paged_shared(c.q, *c.cache, c.table, c.n, starts, shared, lse=lse, **c.kw)

    graphs = []
    for _ in range(2):
        graph, mine = torch.cuda.CUDAGraph(), torch.zeros_like(lse)
        with torch.cuda.graph(graph):
            out = step(mine)
        graphs.append((graph, out, mine))
    lens = list(c.lens)
    for i, (now, st, sh) in enumerate(((lens, c.starts, c.shared), ([n - 20 for n in lens], [0, 6, 9], [400, 128]),
                                       ([0] * 6 + lens[6:], [0, 4, 9], [0, 256]), (lens, [0, 6, 9], [256, 256]))):
        if st == [0, 4, 9]:
            st = [0, 6, 9]
        c.n.copy_(c.ints(now))
        starts.copy_(c.ints(st))
        shared.copy_(c.ints(sh))
        want = step(lse)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, mine in graphs:
            assert torch.equal(out, want) and torch.equal(mine, lse), i
        c.check(want, lse, lens=[max(n, 0) for n in now])


def test_empty_batch(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = Case(torch, cuda, "bf16", 4, 2, 16, [256], [[40, 7]])
    out = fg.decode_flash_gqa_paged_shared(c.q[:0], *c.cache, c.table[:0], c.n[:0], c.ints([0]), c.ints([]).reshape(0))
    assert out.shape == (0, 4, 128)


def test_forked_samples(cuda):
    """As a server runs them: a prompt's queries and keys normalised and rotated, its pages forked to
    samples, tokens appended for some steps, each decoded with the prompt read once, the
    cache compacted, all against the plain paged decode and float64."""
    import torch
    import cuda_llm_ops_amd as fg
    g = torch.Generator(device="cpu").manual_seed(3)
    H, G, P, W, N = 2, 4, 16, 40, 9
    prompt = 333
    kc, vc = (torch.zeros(200, P, H, D, dtype=torch.int8, device=cuda) for _ in range(2))
    scales = dict(k_scale=torch.ones(200, H, device=cuda), v_scale=torch.ones(200, H, device=cuda))
    w = [(1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(cuda) for _ in range(2)]
    inv_freq = (1e4 ** (-torch.arange(0, D, 2) / D)).float().to(cuda)

    def tokens(B, n, first):
        q, k, v = (torch.randn(B, n, h, D, generator=g).to(torch.bfloat16).to(cuda) for h in (H * G, H, H))
        pos = (first[:, None] + torch.arange(n, device=cuda)).to(torch.int32)
        q, k = fg.qk_norm_rope(q, k, pos, inv_freq, *w)
        return q, k, v

    lens = torch.zeros(1, dtype=torch.int32, device=cuda)
    table, lens, _ = fg.fork_kv_paged(kc, vc, torch.full((1, W), -1, dtype=torch.int32, device=cuda), lens,
                                      new_lens=torch.tensor([prompt], dtype=torch.int32, device=cuda), **scales)
    _, k, v = tokens(1, prompt, lens)
    fg.append_kv_paged(k, v, kc, vc, table, lens, **scales)
    lens = lens + prompt
    parents = torch.zeros(N, dtype=torch.int32, device=cuda)
    one = torch.ones(N, dtype=torch.int32, device=cuda)
    starts, shared = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, N], [prompt]))
    for step in range(12):
        table, lens, left = fg.fork_kv_paged(kc, vc, table, lens, parents=parents, new_lens=one, **scales)
        assert int(left) > 0
        q, k, v = tokens(N, 1, lens)
        fg.append_kv_paged(k, v, kc, vc, table, lens, **scales)
        lens = lens + 1
        if step == 5:
            table, used = fg.compact_kv_paged(kc, vc, table, lens, **scales)
            assert int(used) == prompt // P + N * (1 if (prompt % P) + 6 <= P else 2)
        lse = [torch.empty(N, H * G, device=cuda) for _ in range(2)]
        args = (q[:, 0], kc, vc, table, lens)
        out = fg.decode_flash_gqa_paged_shared(*args, starts, shared, lse=lse[0], **scales)
        plain = fg.decode_flash_gqa_paged(*args, lse=lse[1], **scales)
        # (both round to bf16; weights of the shared tokens do too: 2^-8 of sum p |v|, here below 4)
        assert float((out.float() - plain.float()).abs().max()) <= 2.0 ** -8 * 4 * 2
        assert float((lse[0] - lse[1]).abs().max()) <= 2.0 ** -16
        # samples that end are replaced by others'
        parents = torch.tensor([(i * 7 + step) % N if step % 3 == 2 else i for i in range(N)], dtype=torch.int32, device=cuda)
