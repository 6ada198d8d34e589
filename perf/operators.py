"""The paged 8-bit KV cache's operators, each timed through its public entry point.

Writing tokens to the cache (``append``), single-token attention over it
(``decode``), the attention weight that each cached token gets (``weights``)
and the eviction of those that got least (``evict``).  A cache block is one page
of one KV head; 8-bit blocks hold codes (e4m3 or int8) and one fp32 scale.

``run`` computes them in plain torch operations in 32 bits, or (``own``) by the
library's kernels; ``exact`` computes them in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
D = 128
DTYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}

# The ranges that the listed cases stand for (`draw` takes sizes from them).
# (query heads, KV heads) of a layer or of one tensor-parallel shard of it.
HEADS = ((16, 2), (32, 8), (64, 8), (128, 8), (16, 1), (8, 8), (28, 4))
PAGES = (16, 16, 32, 64, 128)
MAX_TOKEN_HEADS = 1 << 22         # padded tokens times KV heads of a drawn case


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One step of a busy server: a new token for each of 64 conversations.
        dict(name="append_step", kind="append", dtype="e4m3", B=64, N=1, S=4096, Hkv=8, page=64, lens_seed=1),
        # Prompts of chat length joining short histories, ragged.
        dict(name="append_chat", kind="append", dtype="int8", B=6, N=777, S=500, Hkv=8, page=16, lens_seed=2),
        # Two long prompts.
        dict(name="append_long", kind="append", dtype="e4m3", B=2, N=16384, S=64, Hkv=8, page=64, lens_seed=3),
        # Two short conversations on one shard of a model: latency only.
        dict(name="decode_tiny", kind="decode", dtype="int8", B=2, S=512, Hq=16, Hkv=2, page=16, lens_seed=4),
        # A lightly loaded server: a few sequences of different lengths.
        dict(name="decode_light", kind="decode", dtype="int8", B=8, S=6000, Hq=32, Hkv=8, page=16, lens_seed=5),
        # A fully loaded server, ragged up to 32K tokens: the largest case.
        dict(name="decode_full", kind="decode", dtype="e4m3", B=64, S=32768, Hq=64, Hkv=8, page=64, lens_seed=6),
        # One user with a long context in a bf16 cache.
        dict(name="weights_one", kind="weights", dtype="bf16", B=1, S=8192, Hq=28, Hkv=4, page=16, lens_seed=7),
        # A loaded server's step.
        dict(name="weights_step", kind="weights", dtype="int8", B=24, S=8192, Hq=32, Hkv=8, page=32, lens_seed=8),
        # A fully loaded one.
        dict(name="weights_full", kind="weights", dtype="e4m3", B=64, S=16384, Hq=64, Hkv=8, page=64, lens_seed=9),
        # Short conversations cut to a small budget: latency only.
        dict(name="evict_small", kind="evict", dtype="int8", B=2, S=600, Hkv=2, page=16, budget=256, recent=32, lens_seed=10),
        # One long bf16 context cut to an eighth.
        dict(name="evict_one", kind="evict", dtype="bf16", B=1, S=32768, Hkv=8, page=16, budget=4096, recent=128, lens_seed=11),
        # A loaded server's caches cut to half.
        dict(name="evict_full", kind="evict", dtype="e4m3", B=32, S=8192, Hkv=8, page=64, budget=4000, recent=256, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "weights", "evict"))
    dtype = rng.choice(("e4m3", "int8") if kind == "decode" else ("e4m3", "int8", "e4m3", "int8", "bf16"))
    hq, hkv = rng.choice(HEADS)
    case = dict(kind=kind, dtype=dtype, Hkv=hkv, page=rng.choice(PAGES), lens_seed=rng.randrange(1 << 20))
    if kind == "append":
        n = rng.choice((1, _log_int(rng, 2, 8192)))
        s = _log_int(rng, 64, 8192)
        most = min(MAX_TOKEN_HEADS // (s * hkv), (MAX_TOKEN_HEADS // 8) // ((n + 64) * hkv))
        case.update(N=n, S=s, B=max(1, min(_log_int(rng, 1, 128), most)))
        return case
    s = _log_int(rng, 128, 32768)
    case.update(S=s, B=max(1, min(_log_int(rng, 1, 64), MAX_TOKEN_HEADS // (s * hkv))))
    if kind == "evict":
        budget = _log_int(rng, 32, s)
        case.update(budget=budget, recent=rng.choice((0, budget // 16, budget // 4)))
    else:
        case.update(Hq=hq)
    return case


# ------------------------------------------------------------------ sizes
def _lens(case):
    """Tokens of each sequence before the call, from the case's own seed."""
    r = random.Random(case["lens_seed"])
    low = case["S"] // 2 if case["kind"] == "evict" else 1
    return [r.randint(low, case["S"]) for _ in range(case["B"])]


def _new_lens(case):
    """New tokens of each sequence: one, or half of N up to N."""
    r = random.Random(case["lens_seed"] + 1)
    return [r.randint((case["N"] + 1) // 2, case["N"]) for _ in range(case["B"])]


def work(case):
    h, size = case["Hkv"], 2 if case["dtype"] == "bf16" else 1
    scaled = 0 if case["dtype"] == "bf16" else 4   # bytes of a block's scale
    lens = _lens(case)
    if case["kind"] == "append":
        n = sum(_new_lens(case))
        blocks = sum((a + m - 1) // case["page"] - a // case["page"] + 1 for a, m in zip(lens, _new_lens(case)))
        return dict(bytes=n * h * 2 * D * (2 + size) + blocks * h * 2 * scaled, flops=0)
    tokens = sum(lens)
    blocks = sum(-(-n // case["page"]) for n in lens)
    if case["kind"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return dict(bytes=h * (4 * tokens + 2 * kept * 2 * D * size + 8 * kept + 4 * scaled * kept // case["page"]), flops=0)
    rows = case["B"] * case["Hq"]
    if case["kind"] == "decode":
        return dict(bytes=h * 2 * (tokens * D * size + blocks * scaled) + rows * (2 * D * 2 + 4),
                    flops=4 * D * case["Hq"] * tokens)
    return dict(bytes=h * (tokens * (D * size + 8) + blocks * scaled) + rows * (D * 2 + 4),
                flops=2 * D * case["Hq"] * tokens)


# ------------------------------------------------------------------ blocks
def _block_scale(amax, dtype):
    """The smallest power of two that brings amax (fp32) inside the codes' range."""
    m, e = torch.frexp(amax)
    top, shift = (0.875, 9) if dtype == "e4m3" else (127 / 128, 7)   # qmax = top * 2^shift
    e = torch.where(amax > 0, e - shift + (m > top), torch.full_like(e, -126)).clamp(min=-126)
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _finite_abs(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def _codes(x, dtype):
    """Scaled fp32 values -> codes (raw bytes), rounded to nearest even and saturated."""
    if dtype == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.nan_to_num(x, nan=0.0).clamp(-127.0, 127.0).round().to(torch.int8).view(torch.uint8)


def _raw(cache):
    """The cache's storage in a type that every indexing takes."""
    return cache.view(torch.uint8) if cache.element_size() == 1 else cache


def _values(raw, dtype):
    return raw.view(DTYPES[dtype]).to(torch.float32)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _keys(g, *shape):
    """Key- or value-like values [..., Hkv, D]: heads of different size and a few large channels."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    x *= 0.5 + torch.rand(shape[-2:-1] + (1,), generator=g, device=DEV)
    x[..., :: 32] *= 4.0
    return x.to(torch.bfloat16)


def _cache(g, pages, case):
    """(cache, scales) of `pages` full pages; scales None for bf16."""
    P, H, dtype = case["page"], case["Hkv"], case["dtype"]
    cache = torch.empty((pages, P, H, D), device=DEV, dtype=DTYPES[dtype])
    scales = None if dtype == "bf16" else torch.empty((pages, H), device=DEV, dtype=torch.float32)
    step = max(1, (1 << 27) // (P * H * D))
    for p0 in range(0, pages, step):
        x = _keys(g, min(step, pages - p0), P, H, D)
        if dtype == "bf16":
            cache[p0:p0 + step] = x
            continue
        x = x.float()
        scales[p0:p0 + step] = _block_scale(x.abs().amax(dim=(1, 3)), dtype)
        _raw(cache)[p0:p0 + step] = _codes(x / scales[p0:p0 + step, None, :, None], dtype)
    return cache, scales


def _table(g, counts, width, first=0):
    """Block table of `counts` pages a sequence in a random order from page `first` on."""
    perm = (torch.randperm(sum(counts), generator=g, device=DEV) + first).to(torch.int32)
    table = torch.zeros((len(counts), max(1, width)), device=DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    return table


def prepare(case, seed):
    g = _gen(seed)
    B, P, H, kind = case["B"], case["page"], case["Hkv"], case["kind"]
    lens = _lens(case)
    st = dict(case=case, lens=torch.tensor(lens, device=DEV, dtype=torch.int32))
    total = lens
    if kind == "append":
        new = _new_lens(case)
        total = [a + n for a, n in zip(lens, new)]
        st["new_lens"] = torch.tensor(new, device=DEV, dtype=torch.int32)
        st["k_new"], st["v_new"] = _keys(g, B, case["N"], H, D), _keys(g, B, case["N"], H, D)
    counts = [-(-n // P) for n in total]
    width = -(-(case["S"] + case.get("N", 0)) // P)
    st["table"] = _table(g, counts, width)
    pages = sum(counts)
    if kind == "evict":
        kept = [-(-min(n, case["budget"]) // P) for n in lens]
        st["new_table"] = _table(g, kept, -(-case["budget"] // P), pages)
        pages += sum(kept)
        w = torch.exp(2.0 * torch.randn((B, H, case["S"]), generator=g, device=DEV)) * (8.0 / case["S"])
        st["weights"] = torch.where(torch.arange(case["S"], device=DEV) < st["lens"][:, None, None], w, torch.zeros_like(w))
    # (one page more than the sequences use)
    st["k"], st["ks"] = _cache(g, pages + 1, case)
    if kind == "weights":
        st["weights"] = torch.zeros((B, H, case["S"]), device=DEV, dtype=torch.float32)
    else:
        st["v"], st["vs"] = _cache(g, pages + 1, case)
    if kind in ("decode", "weights"):
        st["q"] = torch.randn((B, case["Hq"], D), generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    if kind == "weights":   # as the decode before it gives it
        s = _scores(st)
        st["lse"] = torch.logsumexp(s, dim=3).reshape(B, case["Hq"])
    return st


# ------------------------------------------------------------------ plain forms
def _gathered(st, name):
    """The sequences' keys or values in fp32 [B, Hkv, S', D], S' the table's tokens."""
    raw = _raw(st[name])[st["table"].long()]                         # [B, pages, P, H, D]
    x = _values(raw, st["case"]["dtype"])
    if st[name + "s"] is not None:
        x = x * st[name + "s"][st["table"].long()][:, :, None, :, None]
    B, n, P, H, _ = x.shape
    return x.reshape(B, n * P, H, D).transpose(1, 2).contiguous()


def _scores(st):
    """fp32 [B, Hkv, G, S'], -inf past the sequences' ends."""
    B, Hq, H = st["case"]["B"], st["case"]["Hq"], st["case"]["Hkv"]
    k = _gathered(st, "k").transpose(2, 3).contiguous()
    s = torch.matmul(st["q"].float().reshape(B, H, Hq // H, D), k) * (1.0 / math.sqrt(D))
    hidden = torch.arange(s.shape[3], device=DEV) >= st["lens"][:, None, None, None]
    return s.masked_fill(hidden, -math.inf)


def _plain_decode(st):
    B, Hq = st["case"]["B"], st["case"]["Hq"]
    s = _scores(st)
    m = s.amax(dim=3, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, _gathered(st, "v")) / total
    return o.reshape(B, Hq, D).to(torch.bfloat16), (m + torch.log(total)).reshape(B, Hq)


def _plain_weights(st):
    case = st["case"]
    s = _scores(st)
    p = torch.exp(s - st["lse"].reshape(s.shape[:3])[..., None]).sum(dim=2)
    st["weights"] += p[:, :, :case["S"]]
    return st["weights"]


def _plain_append(st):
    case = st["case"]
    B, N, P, dtype = case["B"], case["N"], case["page"], case["dtype"]
    lens, new = st["lens"].long()[:, None], st["new_lens"].long()[:, None]
    first = lens // P                                                # [B, 1]
    J = (N + P - 2) // P + 1                                         # pages that N tokens touch at most
    at = torch.arange(J * P, device=DEV)[None, :] + first * P - lens  # new token of each row
    is_new, is_old = (at >= 0) & (at < new), at < 0
    page_at = first + torch.arange(J, device=DEV)[None, :]
    used = page_at * P < lens + new
    spare = st["k"].shape[0] - 1                                     # rows without a token rewrite its bytes
    pages = torch.where(used, torch.gather(st["table"].long(), 1, page_at.clamp(max=st["table"].shape[1] - 1)), spare)
    rows = at.clamp(0, N - 1)[:, :, None, None].expand(B, J * P, case["Hkv"], D)
    for name in ("k", "v"):
        raw, scales = _raw(st[name]), st[name + "s"]
        before = raw[pages]                                          # [B, J, P, H, D]
        x = torch.gather(st[name + "_new"], 1, rows).reshape(before.shape)
        fresh = is_new.reshape(B, J, P, 1, 1)
        held = (is_old & (lens > 0)).reshape(B, J, P, 1, 1) & used[:, :, None, None, None]
        if scales is None:
            raw[pages] = torch.where(fresh, x, before)
            continue
        x = x.float()
        amax = torch.where(fresh, _finite_abs(x), torch.zeros_like(x)).amax(dim=(2, 4))
        old = scales[pages]
        scale = _block_scale(amax, dtype)
        scale = torch.where(held.any(dim=2)[..., 0], torch.maximum(scale, old), scale)
        moved = _codes(_values(before, dtype) * old[:, :, None, :, None] / scale[:, :, None, :, None], dtype)
        fresh_codes = _codes(x / scale[:, :, None, :, None], dtype)
        raw[pages] = torch.where(fresh, fresh_codes, torch.where(held, moved, before))
        scales[pages] = torch.where(used[:, :, None], scale, old)
    return _cache_out(st)


def _cache_out(st):
    """The cache as it stands: e4m3 codes as numbers, scales beside them."""
    out = dict(k=st["k"], v=st["v"])
    if st["ks"] is not None:
        out.update(k_scale=st["ks"], v_scale=st["vs"])
    return out


def _plain_evict(st):
    case = st["case"]
    B, H, S, P, dtype = case["B"], case["Hkv"], case["S"], case["page"], case["dtype"]
    budget, recent = case["budget"], min(case["recent"], case["budget"])
    lens = st["lens"].long()[:, None, None]
    at = torch.arange(S, device=DEV)[None, None, :]
    # recent tokens before all others, missing ones last; equal weights in order
    rank = torch.where(at < lens, st["weights"], torch.full_like(st["weights"], -math.inf))
    rank = torch.where((at < lens) & (at >= lens - recent), torch.full_like(rank, math.inf), rank)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :budget]
    C = order.shape[2]
    count = lens.clamp(max=budget)
    order = torch.where(torch.arange(C, device=DEV) < count, order, S)
    kept = torch.sort(order, dim=2).values                           # [B, H, C], S where there is none
    there = kept < S
    kept = torch.where(there, kept, 0)
    new_weights = torch.zeros_like(st["weights"])
    new_weights[:, :, :C] = torch.where(there, torch.gather(st["weights"], 2, kept), 0.0)
    table = st["table"].long()
    src_page = torch.gather(table[:, None, :].expand(B, H, table.shape[1]), 2, kept // P)
    heads = torch.arange(H, device=DEV)[None, :, None]
    J = -(-C // P)
    pad = J * P - C
    spare = st["k"].shape[0] - 1
    used = torch.arange(J, device=DEV)[None, :] * P < count[:, :, 0]
    new_pages = torch.where(used, st["new_table"].long()[:, :J], spare)
    rows = torch.nn.functional.pad(there, (0, pad)).reshape(B, H, J, P).permute(0, 2, 3, 1)[..., None]
    for name in ("k", "v"):
        raw, scales = _raw(st[name]), st[name + "s"]
        x = raw[src_page, kept % P, heads]                           # [B, H, C, D]
        before = raw[new_pages]                                      # [B, J, P, H, D]
        if scales is not None:
            x = _values(x, dtype) * scales[src_page, heads][..., None]
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(B, H, J, P, D).permute(0, 2, 3, 1, 4)
        if scales is None:
            raw[new_pages] = torch.where(rows, x, before)
            continue
        amax = torch.where(rows, _finite_abs(x), torch.zeros_like(x)).amax(dim=(2, 4))
        scale = torch.where(used[:, :, None], _block_scale(amax, dtype), scales[new_pages])
        raw[new_pages] = torch.where(rows, _codes(x / scale[:, :, None, :, None], dtype), before)
        scales[new_pages] = scale
    new_lens = st["lens"].clamp(max=budget)
    kept = torch.nn.functional.pad(torch.where(there, kept, -1), (0, budget - C), value=-1).to(torch.int32)
    return dict(_cache_out(st), lens=new_lens, weights=new_weights, kept=kept)


# ------------------------------------------------------------------ the library's calls
def _own(st):
    import cuda_llm_ops_amd as fg
    case = st["case"]
    kind = case["kind"]
    scales = {} if st["ks"] is None else dict(k_scale=st["ks"])
    if kind != "weights" and st["ks"] is not None:
        scales["v_scale"] = st["vs"]
    if kind == "append":
        fg.append_kv_paged(st["k_new"], st["v_new"], st["k"], st["v"], st["table"], st["lens"], new_lens=st["new_lens"],
                           **scales)
        return _cache_out(st)
    if kind == "decode":
        lse = torch.empty((case["B"], case["Hq"]), device=DEV, dtype=torch.float32)
        o = fg.decode_flash_gqa_paged(st["q"], st["k"], st["v"], st["table"], st["lens"], lse=lse, max_seqlen=case["S"],
                                      **scales)
        return o, lse
    if kind == "weights":
        return fg.accumulate_kv_weights_paged(st["q"], st["k"], st["lse"], st["table"], st["lens"], st["weights"],
                                              max_seqlen=case["S"], **scales)
    lens, weights, kept = fg.evict_kv_paged(st["k"], st["v"], st["table"], st["lens"], st["weights"], st["new_table"],
                                            budget=case["budget"], recent=case["recent"], max_seqlen=case["S"], **scales)
    return dict(_cache_out(st), lens=lens, weights=weights, kept=kept)


def run(st):
    if own:
        return _own(st)
    return {"append": _plain_append, "decode": _plain_decode, "weights": _plain_weights,
            "evict": _plain_evict}[st["case"]["kind"]](st)


# ------------------------------------------------------------------ 64 bits
def _exact_rows(st, name, b, n):
    """Sequence b's n keys or values in float64 [n, Hkv, D]."""
    P = st["case"]["page"]
    pages = st["table"][b, :-(-n // P)].long()
    x = _raw(st[name])[pages].view(DTYPES[st["case"]["dtype"]]).double()
    if st[name + "s"] is not None:
        x *= st[name + "s"][pages].double()[:, None, :, None]
    return x.reshape(-1, x.shape[2], D)[:n]


def _exact_attention(st):
    case = st["case"]
    G = case["Hq"] // case["Hkv"]
    o = torch.zeros((case["B"], case["Hq"], D), device=DEV, dtype=torch.float64)
    lse = torch.full((case["B"], case["Hq"]), -math.inf, device=DEV, dtype=torch.float64)
    weights = torch.zeros((case["B"], case["Hkv"], case["S"]), device=DEV, dtype=torch.float64)
    for b, n in enumerate(_lens(case)):
        k = _exact_rows(st, "k", b, n)
        v = _exact_rows(st, "v", b, n) if case["kind"] == "decode" else None
        for h in range(case["Hkv"]):
            rows = slice(h * G, (h + 1) * G)
            s = st["q"][b, rows].double() @ k[:, h].t().contiguous() / math.sqrt(D)
            if v is None:
                weights[b, h, :n] = torch.exp(s - st["lse"][b, rows].double()[:, None]).sum(dim=0)
                continue
            lse[b, rows] = torch.logsumexp(s, dim=1)
            o[b, rows] = torch.softmax(s, dim=1) @ v[:, h].contiguous()
    return weights if case["kind"] == "weights" else (o, lse)


def _exact_block(x, dtype, least):
    """Rows x [n, D] in float64 -> (their codes as float64, the block's scale, at least `least`)."""
    top = float(x[torch.isfinite(x)].abs().max()) if x.numel() else 0.0
    scale = 2.0 ** -126
    while scale * QMAX[dtype] < top:
        scale *= 2.0
    scale = max(scale, least)
    y = (x / scale).clamp(-QMAX[dtype], QMAX[dtype])
    if dtype == "int8":
        return torch.round(y), scale
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # of e4m3 at y; exact for powers of two
    return torch.round(y / step) * step, scale


def exact(case, seed):
    kind = case["kind"]
    # append and evict give whole codes and powers of two: their 64-bit values are worked out on small cases block by block
    if kind in ("append", "evict") and (case["B"] * case["Hkv"] * (case.get("N", 0) + case["S"] // 4) // case["page"] > 4200):
        return None
    st = prepare(case, seed)
    if kind in ("decode", "weights"):
        return _exact_attention(st)
    P, H, dtype = case["page"], case["Hkv"], case["dtype"]
    caches = {n: st[n].view(DTYPES[dtype]).double().cpu() for n in ("k", "v")}
    scales = {n: None if st[n + "s"] is None else st[n + "s"].double().cpu() for n in ("k", "v")}
    old = {n: caches[n].clone() for n in caches}
    old_scales = {n: None if scales[n] is None else scales[n].clone() for n in scales}
    table, out = st["table"].cpu(), {}

    def put(name, page, h, slots, rows, least=0.0):
        """Writes rows [n, D] (float64 values) to slots of a block."""
        if scales[name] is None:
            caches[name][page, slots, h] = rows
            return
        caches[name][page, slots, h], scales[name][page, h] = _exact_block(rows, dtype, least)

    def value(name, page, slots, h):
        x = old[name][page, slots, h]
        return x if old_scales[name] is None else x * old_scales[name][page, h]

    if kind == "append":
        new = {n: st[n + "_new"].double().cpu() for n in ("k", "v")}
        for b, (a, n) in enumerate(zip(_lens(case), _new_lens(case))):
            for j in range(a // P, (a + n - 1) // P + 1):
                page, t0, t1 = int(table[b, j]), max(a, j * P), min(a + n, (j + 1) * P)
                for name in ("k", "v"):
                    for h in range(H):
                        rows, first, least = new[name][b, t0 - a:t1 - a, h], t0 - j * P, 0.0
                        if first > 0 and scales[name] is not None:   # the block's older tokens and scale
                            rows = torch.cat((value(name, page, slice(0, first), h), rows))
                            least, first = float(old_scales[name][page, h]), 0
                        put(name, page, h, slice(first, t1 - j * P), rows, least)
    else:
        w, C = st["weights"].double().cpu(), case["budget"]
        wl = w.tolist()
        out = dict(lens=None, weights=torch.zeros_like(w), kept=None)
        for b, n in enumerate(_lens(case)):
            c = min(n, C)
            near = min(case["recent"], c) if n > C else n
            for h in range(H):
                by_weight = sorted(range(n - near), key=lambda i: (-wl[b][h][i], i))[:c - near]
                kept = torch.tensor(sorted(by_weight) + list(range(n - near, n)))
                out["weights"][b, h, :c] = w[b, h, kept]
                for j in range(-(-c // P)):
                    ids = kept[j * P:(j + 1) * P]
                    for name in ("k", "v"):
                        page = table[b][ids // P].long()
                        rows = old[name][page, ids % P, h]
                        if scales[name] is not None:
                            rows = rows * old_scales[name][page, h][:, None]
                        put(name, int(st["new_table"][b, j]), h, slice(0, len(ids)), rows)
    whole = dtype == "int8"
    out.update(k=None if whole else caches["k"], v=None if whole else caches["v"])
    if scales["k"] is not None:
        out.update(k_scale=scales["k"], v_scale=scales["v"])
    return out
