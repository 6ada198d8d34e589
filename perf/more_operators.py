"""Operators around the library's attention, each timed through its public entry point.

Queries and keys normalised for each head and rotated to their positions, of one
axis or several (``rope``), and the gradients of that (``rope_grad``);
single-token attention for sequences that share the beginning of their caches
(``shared``); the pages of a paged cache forked and freed (``fork``) and moved
together (``compact``).

``run`` computes them in plain torch operations in 32 bits (angles in 64), or
(``own``) by the library's kernels; ``exact`` computes them in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
D = 128                           # head dim of the caches
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}

# The ranges that the listed cases stand for (`draw` takes sizes from them).
# (query heads, KV heads) of a layer or of one tensor-parallel shard of it.
HEADS = ((16, 2), (32, 8), (64, 8), (128, 8), (16, 1), (8, 8), (28, 4))
HEAD_DIMS = (64, 80, 96, 128, 128, 128, 192, 256)
PAGES = (16, 16, 32, 64, 128)
MAX_ROPE = 9 << 23                # elements of q and k of a drawn case
MAX_SHARED_FLOPS = 1 << 37
MAX_CACHE = 1 << 30               # bytes of K of a drawn case's cache


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One step of a busy server: a new token for each of 64 conversations.
        dict(name="rope_step", kind="rope", B=64, S=0, Hq=64, Hkv=8, D=128, R=128, axes="one", norm=True,
             interleaved=False, far=32768, pos64=False),
        # A prompt, q and k as they lie in the fused projection's output.
        dict(name="rope_prompt", kind="rope", B=1, S=4096, Hq=32, Hkv=8, D=128, R=128, axes="one", norm=True,
             interleaved=False, far=0, pos64=True),
        # Prompts of text and pictures: three axes, an odd length.
        dict(name="rope_pictures", kind="rope", B=4, S=6001, Hq=28, Hkv=4, D=128, R=128, axes="sections", norm=True,
             interleaved=False, far=0, pos64=True),
        # A training step's micro-batch.
        dict(name="rope_grad_text", kind="rope_grad", B=2, S=2048, Hq=16, Hkv=2, D=128, R=128, axes="one", norm=True,
             interleaved=False, far=0, pos64=True),
        # One of text and pictures, the axes' frequencies in turn, neighbours paired.
        dict(name="rope_grad_pictures", kind="rope_grad", B=3, S=5003, Hq=32, Hkv=8, D=128, R=128, axes="turns", norm=True,
             interleaved=True, far=0, pos64=True),
        # Eight samples of one prompt on one shard of a model: latency counts.
        dict(name="shared_samples", kind="shared", dtype="int8", Hq=16, Hkv=2, page=16, groups=1, size=8, alone=0,
             shared=2000, own=100, lens_seed=1),
        # A server: four prompts of 16 samples each, and a few conversations of their own.
        dict(name="shared_server", kind="shared", dtype="e4m3", Hq=64, Hkv=8, page=64, groups=4, size=16, alone=5,
             shared=8000, own=1000, lens_seed=2),
        # One long document and 128 questions: the largest case.
        dict(name="shared_document", kind="shared", dtype="bf16", Hq=64, Hkv=8, page=64, groups=1, size=128, alone=0,
             shared=32768, own=1500, lens_seed=3),
        # A step of a beam search: 4 beams of each of 4 prompts go on from their best.
        dict(name="fork_beams", kind="fork", dtype="bf16", Hkv=2, page=16, B=16, N=16, S=700, new=1, spare=40,
             parents="beams", lens_seed=4),
        # 16 samples of each of 16 prompts, with room for 300 tokens.
        dict(name="fork_samples", kind="fork", dtype="e4m3", Hkv=8, page=64, B=16, N=256, S=8000, new=300, spare=100,
             parents="samples", lens_seed=5),
        # A small cache with holes of finished conversations.
        dict(name="compact_small", kind="compact", dtype="int8", Hkv=2, page=16, B=8, S=600, spare=300, lens_seed=6),
        # A server's cache, half of it holes.
        dict(name="compact_server", kind="compact", dtype="bf16", Hkv=8, page=64, B=48, S=8000, spare=3000, lens_seed=7),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope", "rope_grad", "shared", "shared", "fork", "compact"))
    hq, hkv = rng.choice(HEADS)
    if kind in ("rope", "rope_grad"):
        d = rng.choice(HEAD_DIMS)
        per = (hq + hkv) * d
        tokens = min(_log_int(rng, 1, 65536), MAX_ROPE // per)
        b = _log_int(rng, 1, max(1, min(64, tokens)))
        axes = rng.choice(("one", "one", "sections", "turns"))
        return dict(kind=kind, B=b, S=rng.choice((0, 1)) if b == tokens else max(1, tokens // b), Hq=hq, Hkv=hkv, D=d,
                    R=d if rng.random() < 0.7 else 16 * rng.randint(1, d // 16), axes=axes, norm=rng.random() < 0.8,
                    interleaved=rng.random() < 0.4, far=rng.choice((0, 0, 32768, 1 << 20)) if axes == "one" else 0,
                    pos64=rng.random() < 0.5)
    case = dict(kind=kind, dtype=rng.choice(("bf16", "e4m3", "int8")), Hkv=hkv, page=rng.choice(PAGES),
                lens_seed=rng.randrange(1 << 20))
    row = hkv * D * (2 if case["dtype"] == "bf16" else 1)      # bytes of a cached token's K
    if kind == "shared":
        shared, near = _log_int(rng, 64, 32768), _log_int(rng, 1, 2048)
        groups, size, alone = _log_int(rng, 1, 8), _log_int(rng, 2, 128), rng.choice((0, 0, 1, 7))
        most = MAX_SHARED_FLOPS // (4 * D * hq * (shared + near))
        groups = max(1, min(groups, most // 4))
        size = max(2, min(size, most // groups - alone))
        case.update(Hq=hq, groups=groups, size=size, alone=alone, shared=shared, own=near)
        return case
    s = _log_int(rng, 64, 16384)
    case.update(S=s, B=max(1, min(_log_int(rng, 1, 64), MAX_CACHE // (2 * s * row))))
    if kind == "compact":
        case.update(spare=_log_int(rng, 4, max(5, min(4000, MAX_CACHE // (2 * case["page"] * row)))))
        return case
    new = rng.choice((0, 1, _log_int(rng, 2, 500)))
    most = MAX_CACHE // (2 * (new + 2 * case["page"]) * row)
    case.update(N=max(1, min(_log_int(rng, 1, 256), most)), new=new, spare=rng.choice((0, 3, 100)),
                parents=rng.choice(("beams", "samples", "any")))
    return case


# ------------------------------------------------------------------ sizes
def _lens(case):
    """Tokens of each sequence (of a shared case: those of its own), from the case's own seed."""
    r = random.Random(case["lens_seed"])
    if case["kind"] == "shared":
        n = case["groups"] * case["size"] + case["alone"]
        return [r.randint(1, case["own"]) for _ in range(n)]
    return [r.randint(max(1, case["S"] // 4), case["S"]) for _ in range(case["B"])]


def _shared_lens(case):
    r = random.Random(case["lens_seed"] + 1)
    return [r.randint((case["shared"] + 1) // 2, case["shared"]) if case["groups"] > 1 else case["shared"]
            for _ in range(case["groups"])]


def _parents(case):
    """The old row that each new one goes on from (-1: an empty one)."""
    r = random.Random(case["lens_seed"] + 2)
    B, N = case["B"], case["N"]
    if case["parents"] == "samples":
        return [i * B // N for i in range(N)]
    if case["parents"] == "beams":     # of groups of four old rows, mostly the first ones
        return [min(B - 1, i * B // N // 4 * 4 + min(r.randrange(4), r.randrange(4))) for i in range(N)]
    return [r.randrange(-1, B) for _ in range(N)]


def _new_lens(case):
    r = random.Random(case["lens_seed"] + 3)
    return [r.randint(case["new"] // 2, case["new"]) for _ in range(case["N"])]


def _tokens(case):
    return case["B"] * max(1, case["S"])


def _elem(case):
    return 2 if case["dtype"] == "bf16" else 1


def _page_bytes(case, slots):
    """Bytes of `slots` of a page of K and V, and its scales."""
    return 2 * case["Hkv"] * (slots * D * _elem(case) + (0 if case["dtype"] == "bf16" else 4))


def work(case):
    kind = case["kind"]
    if kind in ("rope", "rope_grad"):
        n = _tokens(case) * (case["Hq"] + case["Hkv"]) * case["D"]
        passes = 2 if kind == "rope" else 3 if case["norm"] else 2
        small = _tokens(case) * (8 if case["pos64"] else 4) * (1 if case["axes"] == "one" else 3) + 2 * case["R"]
        if case["norm"]:
            small += 2 * case["D"] * (2 if kind == "rope" else 6)
        return dict(bytes=2 * n * passes + small, flops=n * (8 if kind == "rope" else 16))
    if kind == "shared":
        lens, shared = _lens(case), _shared_lens(case)
        tokens = sum(lens) + sum(shared)
        attended = sum(lens) + case["size"] * sum(shared)
        scales = 0 if case["dtype"] == "bf16" else 8 * case["Hkv"] * tokens // case["page"]
        return dict(bytes=2 * case["Hkv"] * D * _elem(case) * tokens + scales + len(lens) * case["Hq"] * (4 * D + 4),
                    flops=4 * D * case["Hq"] * attended)
    P, lens = case["page"], _lens(case)
    if kind == "fork":
        width = _width(case)
        parents = _parents(case)
        copies = [lens[p] % P for i, p in enumerate(parents) if p >= 0 and lens[p] % P and p in parents[:i]]
        return dict(bytes=4 * (case["B"] + case["N"]) * width + sum(2 * _page_bytes(case, n) for n in copies), flops=0)
    pages = sum(-(-n // P) for n in lens)
    moved = pages * case["spare"] // (pages + case["spare"])     # (of pages in a random order)
    return dict(bytes=8 * case["B"] * _width(case) + 2 * moved * _page_bytes(case, P), flops=0)


def _width(case):
    """Pages of a block table's row."""
    return -(-(case["S"] + case.get("new", 0)) // case["page"])


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _heads(g, *shape):
    """Query-, key- or value-like values [..., heads, D]: heads of different size and a few large channels."""
    x = _randn(g, *shape)
    x *= 0.5 + torch.rand(shape[-2:-1] + (1,), generator=g, device=DEV)
    x[..., :: 32] *= 4.0
    return x.to(torch.bfloat16)


def _positions(case, g):
    """Positions [B, S] or [B], or, of three axes, [3, B, S] or [3, B]: text, then a picture's rows and columns, then text."""
    B, S = case["B"], case["S"]
    dtype = torch.int64 if case["pos64"] else torch.int32
    n = max(1, S)
    if case["axes"] == "one":
        first = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device=DEV)
        pos = first + torch.arange(n, device=DEV)
    else:
        at = torch.arange(n, device=DEV)
        begin, side = n // 8, max(1, int(math.sqrt(n * 0.7)))
        inside = (at >= begin) & (at < begin + side * side)
        rel = (at - begin).clamp(min=0)
        after = begin + side + (at - begin - side * side)
        text = torch.where(at < begin, at, after)
        axes = [torch.where(inside, x, text) for x in (torch.full_like(at, begin), begin + rel // side, begin + rel % side)]
        pos = torch.stack(axes)[:, None, :] + torch.randint(0, 100, (1, B, 1), generator=g, device=DEV)
    return (pos if S > 0 else pos[..., 0]).to(dtype).contiguous()


def _axes_of(case):
    half = case["R"] // 2
    if case["axes"] == "turns":
        return torch.arange(half, device=DEV, dtype=torch.int32) % 3
    t = max(1, half // 4)             # time, then height and width
    h = (half - t + 1) // 2
    return torch.tensor([0] * t + [1] * h + [2] * (half - t - h), device=DEV, dtype=torch.int32)


def _prepare_rope(case, seed):
    g = _gen(seed)
    B, S, Hq, Hkv, d = case["B"], case["S"], case["Hq"], case["Hkv"], case["D"]
    lead = (B, S) if S > 0 else (B,)
    qkv = _heads(g, *lead, Hq + 2 * Hkv, d)
    st = dict(case=case, q=qkv[..., :Hq, :], k=qkv[..., Hq:Hq + Hkv, :], positions=_positions(case, g))
    st["inv_freq"] = (1e6 ** (-torch.arange(0, case["R"], 2, device=DEV, dtype=torch.float64) / case["R"])).float()
    st["axes"] = None if case["axes"] == "one" else _axes_of(case)
    for n in ("q_weight", "k_weight"):
        st[n] = (1.0 + 0.3 * _randn(g, d)).to(torch.bfloat16) if case["norm"] else None
    if case["kind"] == "rope_grad":
        st["grad_q"], st["grad_k"] = (0.05 * _randn(g, *lead, h, d).to(torch.bfloat16) for h in (Hq, Hkv))
    return st


def _cache(g, pages, case):
    """(cache, scales) of `pages` full pages; scales None for bf16."""
    P, H, dtype = case["page"], case["Hkv"], case["dtype"]
    cache = torch.empty((pages, P, H, D), device=DEV, dtype=DTYPES[dtype])
    scales = None if dtype == "bf16" else torch.empty((pages, H), device=DEV, dtype=torch.float32)
    step = max(1, (1 << 27) // (P * H * D))
    for p0 in range(0, pages, step):
        x = _heads(g, min(step, pages - p0), P, H, D)
        if dtype == "bf16":
            cache[p0:p0 + step] = x
            continue
        x = x.float()
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(1, 3)) / QMAX[dtype])))
        scales[p0:p0 + step] = s
        x = (x / s[:, None, :, None]).clamp(-QMAX[dtype], QMAX[dtype])
        _raw(cache)[p0:p0 + step] = (x.to(DTYPES[dtype]) if dtype == "e4m3" else x.round().to(torch.int8)).view(torch.uint8)
    return cache, scales


def _raw(cache):
    """The cache's storage in a type that every indexing takes."""
    return cache.view(torch.uint8) if cache.element_size() == 1 else cache


def _int32(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _table(g, counts, width, pages):
    """Block table of `counts` pages a sequence, in a random order out of `pages`; -1 where there is none."""
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(counts), width), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    return table


def _prepare_shared(case, seed):
    g = _gen(seed)
    P, size = case["page"], case["size"]
    near, shared = _lens(case), _shared_lens(case)
    before = [s for s in shared for _ in range(size)] + [0] * case["alone"]
    lens = [a + b for a, b in zip(before, near)]
    # pages of a group's whole shared pages, then each sequence's others
    full = [s // P for s in shared]
    counts = full + [-(-n // P) - a // P for n, a in zip(lens, before)]
    width = -(-(case["shared"] + case["own"]) // P)
    pages = sum(counts) + 1
    parts = _table(g, counts, max(1, max(counts)), pages)
    table = torch.zeros((len(lens), width), device=DEV, dtype=torch.int32)
    for b in range(len(lens)):
        n = b // size if b < case["groups"] * size else None
        at = 0
        if n is not None:
            at = full[n]
            table[b, :at] = parts[n, :at]
        mine = counts[len(full) + b]
        table[b, at:at + mine] = parts[len(full) + b, :mine]
    st = dict(case=case, table=table, lens=_int32(lens), shared=_int32(shared), group_starts=_int32(
        [n * size for n in range(case["groups"] + 1)]), host_lens=lens)
    st["k"], st["ks"] = _cache(g, pages, case)
    st["v"], st["vs"] = _cache(g, pages, case)
    # (the slots of a page that the shared tokens end in are copies)
    for n, s in enumerate(shared):
        if s % P:
            of = table[n * size:(n + 1) * size, s // P].long()
            for name in ("k", "v"):
                _raw(st[name])[of, :s % P] = _raw(st[name])[of[:1], :s % P]
                if st[name + "s"] is not None:
                    st[name + "s"][of] = st[name + "s"][of[:1]]
    st["q"] = _randn(g, len(lens), case["Hq"], D).to(torch.bfloat16)
    return st


def _prepare_pages(case, seed):
    g = _gen(seed)
    P, lens = case["page"], _lens(case)
    counts = [-(-n // P) for n in lens]
    pages = sum(counts) + case["spare"]
    if case["kind"] == "fork":         # enough for all that the new rows need
        pages += case["N"] * (1 + -(-case["new"] // P))
    st = dict(case=case, lens=_int32(lens), table=_table(g, counts, _width(case), pages))
    st["k"], st["ks"] = _cache(g, pages, case)
    st["v"], st["vs"] = _cache(g, pages, case)
    if case["kind"] == "fork":
        st["parents"], st["new_lens"] = _int32(_parents(case)), _int32(_new_lens(case))
    return st


def prepare(case, seed):
    if case["kind"] in ("rope", "rope_grad"):
        return _prepare_rope(case, seed)
    return _prepare_shared(case, seed) if case["kind"] == "shared" else _prepare_pages(case, seed)


# ------------------------------------------------------------------ plain forms
def _plain_angles(st):
    """cos and sin [..., 1, R/2] in fp32."""
    pos = st["positions"].double()
    f = st["inv_freq"].double()
    if st["axes"] is None:
        theta = pos[..., None] * f
    else:
        theta = torch.gather(pos.movedim(0, -1), -1, st["axes"].long().expand(pos.shape[1:] + f.shape)) * f
    return torch.cos(theta).float()[..., None, :], torch.sin(theta).float()[..., None, :]


def _plain_rotate(x, cos, sin, case):
    """x [..., H, D] rotated (by -theta with -sin)."""
    R = case["R"]
    if case["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
    out = x.clone()
    c, s = a * cos - b * sin, b * cos + a * sin
    if case["interleaved"]:
        out[..., 0:R:2], out[..., 1:R:2] = c, s
    else:
        out[..., :R // 2], out[..., R // 2:R] = c, s
    return out


def _plain_rope(st):
    cos, sin = _plain_angles(st)
    out = {}
    for n in ("q", "k"):
        x = st[n].float()
        if st["case"]["norm"]:
            r = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
            x = x * r * st[n + "_weight"].float()
        out[n] = _plain_rotate(x, cos, sin, st["case"]).to(torch.bfloat16)
    return out


def _plain_rope_grad(st):
    cos, sin = _plain_angles(st)
    out = {}
    for n in ("q", "k"):
        g = _plain_rotate(st["grad_" + n].float(), cos, -sin, st["case"])
        if st["case"]["norm"]:
            x, w = st[n].float(), st[n + "_weight"].float()
            r = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
            x = x * r
            out[n + "_weight"] = (g * x).flatten(0, -2).sum(dim=0)
            g = g * w
            g = r * (g - x * (g * x).mean(dim=-1, keepdim=True))
        out[n] = g.to(torch.bfloat16)
    return out


def _rows(st, name, table, n):
    """n tokens of the pages `table` in fp32 [..., Hkv, n, D]."""
    P = st["case"]["page"]
    pages = table[..., :-(-n // P)].long()
    x = _raw(st[name])[pages].view(DTYPES[st["case"]["dtype"]]).float()          # [..., pages, P, H, D]
    if st[name + "s"] is not None:
        x = x * st[name + "s"][pages][..., None, :, None]
    return x.flatten(-4, -3)[..., :n, :, :].transpose(-3, -2).contiguous()


def _plain_shared(st):
    """Each group's scores of its whole shared pages, and of every sequence's other tokens, under one softmax."""
    case = st["case"]
    P, H, size, G = case["page"], case["Hkv"], case["size"], case["Hq"] // case["Hkv"]
    out, lses = [], []
    groups = [(n * size, (n + 1) * size, s // P) for n, s in enumerate(_shared_lens(case))]
    if case["alone"]:
        groups.append((groups[-1][1], len(st["host_lens"]), 0))
    for b0, b1, full in groups:
        n = b1 - b0
        q = st["q"][b0:b1].float().reshape(n, H, G, D)
        most = max(st["host_lens"][b0:b1]) - full * P
        k = _rows(st, "k", st["table"][b0:b1, full:], most).transpose(2, 3).contiguous()
        s = torch.matmul(q, k)
        hidden = torch.arange(most, device=DEV) >= (st["lens"][b0:b1] - full * P)[:, None, None, None]
        s = s.masked_fill(hidden, -math.inf)
        if full:
            k = _rows(st, "k", st["table"][b0], full * P).transpose(1, 2).contiguous()
            first = torch.matmul(q.transpose(0, 1).reshape(H, n * G, D), k)
            s = torch.cat((first.reshape(H, n, G, full * P).transpose(0, 1), s), dim=3)
        s = s * (1.0 / math.sqrt(D))
        m = s.amax(dim=3, keepdim=True)
        p = torch.exp(s - m)
        total = p.sum(dim=3, keepdim=True)
        o = torch.matmul(p[..., full * P:].contiguous(), _rows(st, "v", st["table"][b0:b1, full:], most))
        if full:
            rows = p[..., :full * P].transpose(0, 1).reshape(H, n * G, full * P)
            o = o + torch.matmul(rows, _rows(st, "v", st["table"][b0], full * P)).reshape(H, n, G, D).transpose(0, 1)
        out.append((o / total).reshape(n, H * G, D).to(torch.bfloat16))
        lses.append((m + torch.log(total)).reshape(n, H * G))
    return torch.cat(out), torch.cat(lses)


def _cache_out(st, **more):
    out = dict(k=st["k"], v=st["v"], **more)
    if st["ks"] is not None:
        out.update(k_scale=st["ks"], v_scale=st["vs"])
    return out


def _plain_fork(st):
    case = st["case"]
    P, N, pages = case["page"], case["N"], st["k"].shape[0]
    parents = st["parents"].long()
    there = parents >= 0
    lens = torch.where(there, st["lens"].long()[parents.clamp(min=0)], 0)
    full, part = lens // P, lens % P
    cell = torch.arange(st["table"].shape[1], device=DEV)[None, :]
    old = st["table"].long()[parents.clamp(min=0)]
    # the first row of each parent keeps its last page
    rows = torch.arange(N, device=DEV)
    first = torch.full((case["B"] + 1,), N, device=DEV).scatter_reduce(0, torch.where(there, parents, case["B"]), rows, "amin")
    keeps = there & (first[torch.where(there, parents, case["B"])] == rows)
    kept = (cell < full[:, None]) | ((cell == full[:, None]) & (part > 0)[:, None] & keeps[:, None])
    used = torch.zeros(pages + 1, device=DEV, dtype=torch.bool)
    used[torch.where(kept, old, pages)] = True
    free = torch.nonzero(~used[:pages])[:, 0]
    wanted = (cell < -(-(lens + st["new_lens"]) // P)[:, None]) & ~kept
    rank = (torch.cumsum(wanted.flatten(), 0) - 1).reshape(wanted.shape)
    table = torch.where(kept, old, torch.where(wanted, free[rank.clamp(min=0, max=free.shape[0] - 1)], -1))
    copied = torch.nonzero(there & ~keeps & (part > 0))[:, 0]
    at = full[copied]
    src, dst = old[copied, at], table[copied, at]
    held = (torch.arange(P, device=DEV)[None, :] < part[copied, None])[:, :, None, None]
    for name in ("k", "v"):
        raw = _raw(st[name])
        raw[dst] = torch.where(held, raw[src], raw[dst])
        if st[name + "s"] is not None:
            st[name + "s"][dst] = st[name + "s"][src]
    num_free = (free.shape[0] - wanted.sum()).to(torch.int32).reshape(1)
    return _cache_out(st, table=table.to(torch.int32), lens=lens.to(torch.int32), free=num_free)


def _plain_compact(st):
    case = st["case"]
    P, pages = case["page"], st["k"].shape[0]
    table = st["table"].long()
    cells = torch.arange(table.shape[1], device=DEV)[None, :] < -(-st["lens"].long() // P)[:, None]
    live = torch.zeros(pages + 1, device=DEV, dtype=torch.bool)
    live[torch.where(cells, table, pages)] = True
    live = live[:pages]
    count = live.sum()
    at = torch.arange(pages, device=DEV)
    src, dst = torch.nonzero(live & (at >= count))[:, 0], torch.nonzero(~live & (at < count))[:, 0]
    moved = at.clone()
    moved[src] = dst
    for name in ("k", "v"):
        raw = _raw(st[name])
        raw[dst] = raw[src]
        if st[name + "s"] is not None:
            st[name + "s"][dst] = st[name + "s"][src]
    new = torch.where(cells, moved[table.clamp(min=0)], -1).to(torch.int32)
    return _cache_out(st, table=new, used=count.to(torch.int32).reshape(1))


# ------------------------------------------------------------------ the library's calls
def _own(st):
    import cuda_llm_ops_amd as fg
    case = st["case"]
    kind = case["kind"]
    if kind in ("rope", "rope_grad"):
        how = dict(q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS, axes=st["axes"],
                   interleaved=case["interleaved"])
        if kind == "rope":
            q, k = fg.qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], **how)
            return dict(q=q, k=k)
        q, k, qw, kw = fg.qk_norm_rope_backward(st["grad_q"], st["grad_k"], st["q"], st["k"], st["positions"],
                                                st["inv_freq"], **how)
        return dict(q=q, k=k, q_weight=qw, k_weight=kw) if case["norm"] else dict(q=q, k=k)
    scales = {} if st["ks"] is None else dict(k_scale=st["ks"], v_scale=st["vs"])
    if kind == "shared":
        lse = torch.empty(st["q"].shape[:2], device=DEV, dtype=torch.float32)
        o = fg.decode_flash_gqa_paged_shared(st["q"], st["k"], st["v"], st["table"], st["lens"], st["group_starts"],
                                             st["shared"], lse=lse, **scales)
        return o, lse
    if kind == "fork":
        table, lens, free = fg.fork_kv_paged(st["k"], st["v"], st["table"], st["lens"], parents=st["parents"],
                                             new_lens=st["new_lens"], **scales)
        return _cache_out(st, table=table, lens=lens, free=free)
    table, used = fg.compact_kv_paged(st["k"], st["v"], st["table"], st["lens"], **scales)
    return _cache_out(st, table=table, used=used)


def run(st):
    if own:
        return _own(st)
    return {"rope": _plain_rope, "rope_grad": _plain_rope_grad, "shared": _plain_shared, "fork": _plain_fork,
            "compact": _plain_compact}[st["case"]["kind"]](st)


# ------------------------------------------------------------------ 64 bits
def _exact_turned(x, weight, theta, case):
    """x [T, H, D] in float64 normalised and rotated, as complex numbers times exp(i theta [T, R/2])."""
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(dim=2, keepdim=True) / x.shape[2] + EPS) * weight
    R = case["R"]
    pairs = x[:, :, :R].unflatten(2, (R // 2, 2) if case["interleaved"] else (2, R // 2))
    pairs = pairs if case["interleaved"] else pairs.transpose(2, 3)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(theta), theta)[:, None, :]
    y = torch.view_as_real(z)
    y = y if case["interleaved"] else y.transpose(2, 3)
    return torch.cat((y.flatten(2, 3), x[:, :, R:]), dim=2)


def _exact_rope(case, st):
    lead = st["q"].shape[:-2]
    T, d = _tokens(case), case["D"]
    pos = st["positions"].double().reshape(-1, T)
    axis = torch.zeros(case["R"] // 2, device=DEV, dtype=torch.long) if st["axes"] is None else st["axes"].long()
    grad = case["kind"] == "rope_grad"
    out = {}
    for n, heads in (("q", case["Hq"]), ("k", case["Hkv"])):
        weight = st[n + "_weight"].double().requires_grad_(grad) if case["norm"] else None
        x = st[n].reshape(T, heads, d)
        done = torch.empty((T, heads, d), device=DEV, dtype=torch.float64)
        step = max(1, (1 << 24) // (heads * d))
        for t in range(0, T, step):
            theta = pos[axis, t:t + step].t().contiguous() * st["inv_freq"].double()
            if not grad:
                done[t:t + step] = _exact_turned(x[t:t + step].double(), weight, theta, case)
                continue
            with torch.enable_grad():
                leaf = x[t:t + step].double().requires_grad_(True)
                y = _exact_turned(leaf, weight, theta, case)
                y.backward(st["grad_" + n].reshape(T, heads, d)[t:t + step].double())
            done[t:t + step] = leaf.grad
        out[n] = done.reshape(lead + (heads, d))
        if grad and case["norm"]:
            out[n + "_weight"] = weight.grad
    return out


def _exact_shared(case, st):
    P, G = case["page"], case["Hq"] // case["Hkv"]
    B = len(st["host_lens"])
    o = torch.zeros((B, case["Hq"], D), device=DEV, dtype=torch.float64)
    lse = torch.zeros((B, case["Hq"]), device=DEV, dtype=torch.float64)
    for b, n in enumerate(st["host_lens"]):
        pages = st["table"][b, :-(-n // P)].long()
        kv = []
        for name in ("k", "v"):
            x = _raw(st[name])[pages].view(DTYPES[case["dtype"]]).double()
            if st[name + "s"] is not None:
                x *= st[name + "s"][pages].double()[:, None, :, None]
            kv.append(x.reshape(-1, case["Hkv"], D)[:n])
        for h in range(case["Hkv"]):
            rows = slice(h * G, (h + 1) * G)
            s = st["q"][b, rows].double() @ kv[0][:, h].t().contiguous() / math.sqrt(D)
            lse[b, rows] = torch.logsumexp(s, dim=1)
            o[b, rows] = torch.softmax(s, dim=1) @ kv[1][:, h].contiguous()
    return o, lse


def exact(case, seed):
    # (forking and compacting move bytes and whole numbers)
    if case["kind"] in ("fork", "compact"):
        return None
    st = prepare(case, seed)
    return _exact_shared(case, st) if case["kind"] == "shared" else _exact_rope(case, st)
