"""GPU tests of the paged KV cache's operators against their definitions in
float64 (tests/_kv_reference.py): codes, scales, indices and moved weights bit
for bit, attention and attention weights to bounds worked out from the kernels'
roundings."""
import math

import numpy as np
import pytest

from tests import _kv_reference as ref

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(128)


def _fg():
    import cuda_llm_ops_amd as fg
    return fg


def _torch():
    import torch
    return torch


def _x(rng, *shape):
    """Key-like bf16 values: heads of different size, a few large channels."""
    torch = _torch()
    x = rng.standard_normal(shape).astype(np.float32)
    x *= np.exp2(rng.integers(-3, 4, size=shape[-2:-1] + (1,))).astype(np.float32)
    x[..., ::32] *= 4
    return torch.from_numpy(x).to(torch.bfloat16)


def _table(rng, B, width, pages, first=0):
    """Distinct pages in a random order."""
    return (first + rng.permutation(pages - first)[:B * width].reshape(B, width)).astype(np.int32)


class Cache:
    """K and V caches with scales: on the GPU and as decoded float64 numbers."""

    def __init__(self, cuda, rng, dtype, pages, P, H, pad=0, scales=True):
        torch = _torch()
        self.dtype, self.cuda = dtype, cuda
        self.t, self.s, self.n, self.sn = [], [], [], []
        for _ in range(2):
            # (heads of a wider tensor when pad > 0: strides other than the shape's)
            x = _x(rng, pages, P, H + pad, 128).float().numpy()
            s = None
            if dtype == "bf16":
                full = torch.from_numpy(x).to(torch.bfloat16)
            elif scales:
                s = np.array([[ref.power_scale(np.abs(x[p, :, h]).max(), dtype) for h in range(H + pad)]
                              for p in range(pages)])
                full = self._coded(ref.round_code(x / s[:, None, :, None], dtype))
            else:
                full = self._coded(ref.round_code(x / 0.25, dtype))
            full = full.to(cuda)
            self.t.append(full[:, :, :H])
            self.n.append(ref.numbers(self.t[-1]))
            self.s.append(None if s is None else torch.from_numpy(s.astype(np.float32)).to(cuda)[:, :H])
            self.sn.append(None if s is None else s[:, :H].copy())

    def _coded(self, codes):
        torch = _torch()
        return torch.from_numpy(codes.astype(np.float32)).to(ref.DTYPES[self.dtype])

    @property
    def scales(self):
        if self.s[0] is not None:
            return dict(k_scale=self.s[0], v_scale=self.s[1])
        return dict(k_scale=0.25, v_scale=0.25) if self.dtype == "e4m3" else {}

    def check(self, what):
        for i, name in enumerate("kv"):
            got = ref.numbers(self.t[i])
            assert np.array_equal(got, self.n[i], equal_nan=True), \
                f"{what}: {name} codes differ at {np.argwhere(~((got == self.n[i]) | (np.isnan(got) & np.isnan(self.n[i]))))[:4].tolist()}"
            if self.sn[i] is not None:
                assert np.array_equal(self.s[i].cpu().double().numpy(), self.sn[i]), f"{what}: {name} scales"


def _i32(cuda, a):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(cuda)


def _append(cuda, c, k, v, table, lens, news, what, **kw):
    torch = _torch()
    _fg().append_kv_paged(k.to(cuda), v.to(cuda), c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens),
                          new_lens=None if news is None else _i32(cuda, news), **c.scales)
    torch.cuda.synchronize()
    news = [k.shape[1]] * len(lens) if news is None else news
    for i, x in enumerate((k, v)):
        ref.append(c.n[i], c.sn[i], c.dtype, x.float().numpy().astype(np.float64), table, lens, news, whole=0.25)
    c.check(what)


KINDS = [("bf16", False), ("e4m3", True), ("e4m3", False), ("int8", True)]


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype,scales", KINDS)
@pytest.mark.parametrize("P", [1, 2, 4, 8, 16, 32, 64, 128, 256, 1024])
def test_append_page_sizes(cuda, P, dtype, scales):
    """Empty, short and page-filling histories; no, one and many new tokens;
    starts and ends inside, at and past a page's border."""
    what = f"append P={P} {dtype} scales={scales}"
    print(what, flush=True)
    rng = np.random.default_rng(P)
    lens = [0, 1, P - 1, P, P + 3, 2 * P - 1, 5]
    news = [1, P, 1, 2 * P + 1, 0, 3, 37]
    N = max(news)
    width = -(-(max(lens) + N) // P) + 1
    pages = len(lens) * width + 3
    c = Cache(cuda, rng, dtype, pages, P, 3, scales=scales)
    table = _table(rng, len(lens), width, pages)
    _append(cuda, c, _x(rng, len(lens), N, 3, 128), _x(rng, len(lens), N, 3, 128), table, lens, news, what)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_append_grows_a_block_token_by_token(cuda, dtype):
    """40 single-token calls over a block of 16 and into the next ones, each token
    up to twice the one before: every older code is rounded again as defined."""
    rng = np.random.default_rng(4)
    c = Cache(cuda, rng, dtype, 8, 16, 2)
    table = _table(rng, 2, 4, 8)
    for i in range(40):
        size = 2.0 ** (i % 16) * 1e-3
        k, v = (_x(rng, 2, 1, 2, 128) * size for _ in range(2))
        _append(cuda, c, k, v, table, [i, i + 3], None, f"{dtype} token {i}")


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_append_keeps_scales_that_are_no_powers_of_two(cuda, dtype):
    torch = _torch()
    rng = np.random.default_rng(5)
    c = Cache(cuda, rng, dtype, 4, 16, 2)
    for i in range(2):
        c.s[i] *= 1.37
        c.sn[i] = c.s[i].cpu().double().numpy()
    table = _table(rng, 1, 3, 4)
    _append(cuda, c, _x(rng, 1, 4, 2, 128) * 0.01, _x(rng, 1, 4, 2, 128) * 0.01, table, [7], None, f"{dtype} kept")
    _append(cuda, c, _x(rng, 1, 3, 2, 128) * 1000, _x(rng, 1, 3, 2, 128) * 1000, table, [11], None, f"{dtype} grown")
    assert torch.equal(c.s[0][int(table[0, 0])].cpu().double() % 1, torch.zeros(2, dtype=torch.float64))


@pytest.mark.parametrize("dtype,scales", KINDS[1:])
def test_append_values_at_the_ends_of_the_range(cuda, dtype, scales):
    """Zeros, the smallest and largest bf16 values, every bf16 significand at the
    codes' borders, infinities and NaN, alone in a block and among others."""
    torch = _torch()
    rng = np.random.default_rng(6)
    c = Cache(cuda, rng, dtype, 24, 8, 2, scales=scales)
    table = _table(rng, 2, 11, 24)
    bits = np.zeros((2, 80, 2, 128), dtype=np.uint16)
    every = np.arange(0x3f00, 0x4400, dtype=np.uint16)          # 0.5 to 512
    bits[0, :8, 0] = rng.choice(every, size=(8, 128))
    bits[0, 8:24, :] = rng.integers(0, 0x7f80, size=(16, 2, 128))  # any finite value
    bits[0, 24:32, 0] = 1                                        # the smallest
    bits[0, 32:40, :] = 0x7f7f                                   # the largest
    bits[0, 40:48, 0, ::5] = 0x7f80                              # inf among zeros
    bits[0, 48:56] = rng.choice(every, size=(8, 2, 128))
    bits[0, 48:56, :, 3] = 0x7f80
    bits[0, 48:56, :, 4] = 0xff80
    bits[0, 48:56, :, 5] = 0x7fc0                                # NaN
    bits[0, 56:64] = 0xff80
    bits[0, 64:72] = 0x8000
    bits[1, :] = rng.integers(0x3a00, 0x4480, size=(80, 2, 128))
    k = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16)
    _append(cuda, c, k, -k, table, [0, 3], None, f"{dtype} scales={scales} ends")


@pytest.mark.parametrize("dtype,scales", KINDS)
def test_append_strides_and_pages_outside(cuda, dtype, scales):
    """Heads of wider caches and of a wider qkv tensor; pages -1, num_pages and a
    table that ends before the tokens do."""
    rng = np.random.default_rng(7)
    c = Cache(cuda, rng, dtype, 12, 16, 2, pad=3, scales=scales)
    table = _table(rng, 3, 3, 12)
    table[1, 1] = -1
    table[2, 0] = 12
    qkv = _x(rng, 3, 70, 9, 128)
    k, v = qkv.to(cuda)[:, :, 4:6], qkv.to(cuda)[:, :, 7:9]
    _fg().append_kv_paged(k, v, c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, [3, 0, 9]), **c.scales)
    _torch().cuda.synchronize()
    for i, x in enumerate((qkv[:, :, 4:6], qkv[:, :, 7:9])):
        ref.append(c.n[i], c.sn[i], dtype, x.float().numpy().astype(np.float64), table, [3, 0, 9], [70] * 3, whole=0.25)
    c.check(f"strides {dtype}")


def test_append_lengths_out_of_range(cuda):
    """Negative lengths count as 0, too many new tokens as N, histories past the table write nothing."""
    rng = np.random.default_rng(8)
    c = Cache(cuda, rng, "int8", 20, 4, 1)
    table = _table(rng, 4, 4, 20)
    k, v = _x(rng, 4, 6, 1, 128), _x(rng, 4, 6, 1, 128)
    _append(cuda, c, k, v, table, [-5, 16, 2 ** 31 - 1, 14], [9, 6, 6, -2], "lengths")


def test_append_nothing(cuda):
    torch = _torch()
    rng = np.random.default_rng(9)
    c = Cache(cuda, rng, "e4m3", 4, 16, 2)
    empty = torch.empty((2, 0, 2, 128), dtype=torch.bfloat16)
    _append(cuda, c, empty, empty, _table(rng, 2, 2, 4), [0, 5], None, "no tokens")
    none = torch.empty((0, 3, 2, 128), dtype=torch.bfloat16)
    _append(cuda, c, none, none, np.zeros((0, 2), np.int32), [], None, "no sequences")


# ------------------------------------------------------------------ decode
def _check_decode(c, q, table, lens, got_o, got_lse, what):
    o, lse, mass, err = ref.decode(q.float().numpy().astype(np.float64), c.n[0], c.sn[0], c.n[1], c.sn[1], table, lens,
                                   SCALE)
    got_o, got_lse = got_o.float().cpu().double().numpy(), got_lse.cpu().double().numpy()
    empty = np.isneginf(lse)
    assert np.all(got_o[empty] == 0) and np.array_equal(np.isneginf(got_lse), empty), f"{what}: empty rows"
    # P rounded to fp16 (half a step 2^-11; below 2^-29 of the largest one, 2^-40 of
    # it at most, hence the tokens' share), each P and the sums to fp32 with the
    # scores' errors twice (numerator and denominator); then O to bf16.
    tol = mass * (2.0 ** -11 + 2.2 * err[..., None] + 2.0 ** -24 * 2 * (max(lens) + 40)) + 2.0 ** -8 * np.abs(o)
    tol += 2.0 ** -39 * max(lens) * np.abs(mass).max() + 1e-30
    bad = np.abs(got_o - o) > tol
    assert not bad.any(), f"{what}: O off by {np.abs(got_o - o)[bad].max()} at {np.argwhere(bad)[0].tolist()}"
    d = np.abs(got_lse[~empty] - lse[~empty])
    e = (err + 2.0 ** -24 * (2 * max(lens, default=0) + 40) + 2.0 ** -22 * np.abs(np.where(empty, 0, lse)))[~empty]
    assert np.all(d <= e), f"{what}: lse off by {d.max()}"


def _for_teams(cuda, table, P, H):
    """The block table with room for so many tokens that a decode without a given
    split length shares the batch out over teams, not in splits (more than
    2048 tokens of a head per CU); the entries that no sequence reaches are garbage."""
    cus = _torch().cuda.get_device_properties(cuda).multi_processor_count
    width = (2048 * cus // (len(table) * H) + P) // P
    wide = np.random.default_rng(5).integers(-9, 10 ** 9, size=(len(table), width))
    wide[:, :table.shape[1]] = table
    return wide


def _decode(cuda, c, q, table, lens, what, **kw):
    """One decode, and one over teams where no argument settles the form."""
    torch = _torch()
    tables = [table]
    if not {"split_tokens", "workspace", "max_seqlen"} & kw.keys():
        tables.append(_for_teams(cuda, table, c.t[0].shape[1], c.t[0].shape[2]))
    for form, t in zip(("", " in teams"), tables):
        lse = torch.full(q.shape[:2], float("nan"), dtype=torch.float32, device=cuda)
        o = _fg().decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, t), _i32(cuda, lens), lse=lse,
                                         **c.scales, **kw)
        torch.cuda.synchronize()
        _check_decode(c, q, table, lens, o, lse, what + form)
    return o, lse


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [1, 2, 4, 8, 16, 32, 64, 256, 1024])
def test_decode_page_sizes(cuda, P, dtype):
    what = f"decode P={P} {dtype}"
    print(what, flush=True)
    rng = np.random.default_rng(20 + P)
    lens = [700, 1, 333, 0, 32, 129]
    width = -(-700 // P)
    pages = len(lens) * width + 2
    c = Cache(cuda, rng, dtype, pages, P, 2)
    q = _x(rng, len(lens), 16, 128)
    _decode(cuda, c, q, _table(rng, len(lens), width, pages), lens, what)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("G,H", [(1, 1), (1, 4), (3, 3), (7, 4), (16, 1), (16, 2)])
def test_decode_heads_and_splits(cuda, G, H, dtype):
    what = f"decode G={G} Hkv={H} {dtype}"
    print(what, flush=True)
    rng = np.random.default_rng(40 + G)
    lens = [1200, 0, 129, 640]
    c = Cache(cuda, rng, dtype, 4 * 75 + 1, 16, H)
    table = _table(rng, 4, 75, 4 * 75 + 1)
    q = _x(rng, 4, G * H, 128)
    _decode(cuda, c, q, table, lens, what)
    for split in (128, 512):
        _decode(cuda, c, q, table, lens, f"{what} split={split}", split_tokens=split)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [8, 16, 64])
def test_decode_scales_far_apart(cuda, P, dtype):
    """Blocks of very different scales (K's within what keeps scores ordinary, V's
    over 2^60), rising and falling along the sequence, and scales that are no
    powers of two: the running V scale is raised in every order."""
    torch = _torch()
    rng = np.random.default_rng(60 + P)
    lens = [500, 77]
    width = -(-500 // P)
    pages = 2 * width
    c = Cache(cuda, rng, dtype, pages, P, 2)
    table = _table(rng, 2, width, pages)
    for i, spread in ((0, 2), (1, 30)):
        c.sn[i] = np.float32(c.sn[i] * np.exp2(rng.integers(-spread, spread + 1, size=c.sn[i].shape)) *
                             rng.uniform(0.5, 1.0, size=c.sn[i].shape)).astype(np.float64)
        c.s[i] = torch.from_numpy(c.sn[i].astype(np.float32)).to(cuda)
    _decode(cuda, c, _x(rng, 2, 8, 128), table, lens, f"scales P={P} {dtype}")


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_decode_garbage_outside_the_sequences(cuda, dtype):
    """Codes (NaN among the e4m3 ones) and NaN scales of other pages, slots and
    table entries past the lengths do not matter; entries outside the cache are clamped."""
    torch = _torch()
    rng = np.random.default_rng(70)
    for P in (4, 16, 64):
        lens = [45, 3 * P + 1, 200]
        width = -(-200 // P)
        pages = 3 * width + 4
        c = Cache(cuda, rng, dtype, pages, P, 2)
        table = _table(rng, 3, width, pages)
        q = _x(rng, 3, 8, 128)
        used = np.zeros((pages, P), bool)
        for b, n in enumerate(lens):
            for t in range(n):
                used[table[b, t // P], t % P] = True
        for i in range(2):
            raw = c.t[i].view(torch.uint8)
            raw[torch.from_numpy(~used).to(cuda)] = 0x7f
            c.s[i][torch.from_numpy(~used.any(axis=1)).to(cuda)] = float("nan")
        far = table.copy()
        for b, n in enumerate(lens):
            far[b, -(-n // P):] = (-7, 10 ** 9, pages)[b]
        _decode(cuda, c, q, far, lens, f"garbage P={P} {dtype}")


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("P", [4, 16, 64])
def test_decode_blocks_of_zeros(cuda, P, dtype):
    """Blocks of zeros, whose scale is 2^-126, alone and before and after others."""
    rng = np.random.default_rng(75)
    lens = [200, 3 * P, 150, 1]
    width = -(-200 // P)
    c = Cache(cuda, rng, dtype, 4 * width, P, 2)
    table = _table(rng, 4, width, 4 * width)
    zero = [table[0], table[1][:1], table[2][1:], table[3]]
    for i in range(2):
        for p in np.concatenate(zero):
            c.t[i].view(_torch().uint8)[int(p)] = 0
            c.s[i][int(p)] = 2.0 ** -126
            c.n[i][p] = 0
            c.sn[i][p] = 2.0 ** -126
    o, _ = _decode(cuda, c, _x(rng, 4, 8, 128), table, lens, f"zeros P={P} {dtype}")
    assert not o[0].any() and not o[3].any()


def test_decode_strided_and_prepared(cuda):
    """Wider caches, scales and queries; an output view; a prepared launch."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(80)
    c = Cache(cuda, rng, "int8", 40, 16, 2, pad=1)
    table, lens = _table(rng, 2, 20, 40), [300, 41]
    wide = _x(rng, 2, 24, 128)
    q = wide[:, 8:16]
    out = torch.zeros((2, 24, 128), dtype=torch.bfloat16, device=cuda)
    lse = torch.empty((2, 8), dtype=torch.float32, device=cuda)
    call = fg.prepare_decode_paged(wide.to(cuda)[:, 8:16], c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens),
                                   out=out[:, 8:16], lse=lse, **c.scales)
    assert call() is call.out
    torch.cuda.synchronize()
    _check_decode(c, q, table, lens, out[:, 8:16], lse, "strided")
    assert not out[:, :8].any() and not out[:, 16:].any()


def test_decode_same_bits_as_the_whole_cache_scale(cuda):
    """Equal block scales against the paged fp8 decode of one scale: the same
    mathematics but for P's rounding (2^-11 here, 2^-8 there, half a step each)."""
    torch = _torch()
    rng = np.random.default_rng(81)
    c = Cache(cuda, rng, "e4m3", 80, 16, 4, scales=False)
    table, lens = _i32(cuda, _table(rng, 2, 40, 80)), _i32(cuda, [600, 317])
    q = _x(rng, 2, 16, 128).to(cuda)
    whole = _fg().decode_flash_gqa_paged(q, c.t[0], c.t[1], table, lens, k_scale=0.25, v_scale=0.25)
    s = torch.full((80, 4), 0.25, dtype=torch.float32, device=cuda)
    blocks = _fg().decode_flash_gqa_paged(q, c.t[0], c.t[1], table, lens, k_scale=s, v_scale=s)
    v = 0.25 * c.t[1].float().abs().max()
    assert (whole.float() - blocks.float()).abs().max() <= v * (2.0 ** -8 + 2.0 ** -11) + 2 * 2.0 ** -8 * blocks.float().abs().max()


@pytest.mark.parametrize("form", ["whole", "splits", "teams"])
@pytest.mark.parametrize("P", [4, 16, 64])
def test_decode_scores_of_minus_infinity(cuda, P, form):
    """Keys whose scores overflow to -inf get nothing, wherever they lie; a row of
    such keys alone is NaN, as the formula has it."""
    torch = _torch()
    rng = np.random.default_rng(82)
    width = -(-300 // P)
    c = Cache(cuda, rng, "int8", 2 * width, P, 1)
    table, lens = _table(rng, 2, width, 2 * width), [300, 40]
    alive = np.zeros(300, bool)
    alive[140:150] = alive[299] = True
    # 3e38 * -1 * 64 / sqrt(128) is past fp32's range; the alive keys' products are 0
    raw = c.t[0].view(torch.uint8)
    raw[:, :, 0, 7] = 0xff
    for t in np.flatnonzero(alive):
        raw[int(table[0, t // P]), t % P, 0, 7] = 0
    c.s[0].fill_(64.0)
    q = _x(rng, 2, 2, 128)
    q[:, 0, :] = 0.0
    q[:, 0, 7] = 3e38
    lse = torch.empty((2, 2), device=cuda)
    of = _for_teams(cuda, table, P, 1) if form == "teams" else table
    o = _fg().decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, of), _i32(cuda, lens), lse=lse,
                                     split_tokens=128 if form == "splits" else 0, **c.scales)
    torch.cuda.synchronize()
    v = ref.gather(c.n[1], c.sn[1], table, 0, 300, 0)[alive].mean(axis=0)
    size = np.abs(ref.gather(c.n[1], c.sn[1], table, 0, 300, 0)[alive]).mean(axis=0)
    got = o[0, 0].float().cpu().double().numpy()
    # equal P's of 1 round to nothing; sums of 11 terms and two products in fp32, O to bf16
    assert np.all(np.abs(got - v) <= 2.0 ** -8 * np.abs(v) + 2.0 ** -20 * size)
    assert abs(float(lse[0, 0]) - math.log(11)) <= 2.0 ** -21
    assert bool(o[1, 0].isnan().all())           # no key of row 1 is alive


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("B,H,S", [(1, 8, 640), (1, 8, 641), (3, 1, 5000), (16, 4, 1024), (16, 4, 1025), (64, 8, 130),
                                   (65, 8, 130), (8, 8, 8192), (8, 8, 8200), (300, 1, 40)])
def test_decode_forms(cuda, B, H, S, dtype):
    """Either side of where sequences are split, and shared out over teams: the
    lengths 0, 1 and the longest among them."""
    what = f"decode B={B} Hkv={H} S={S} {dtype}"
    print(what, flush=True)
    rng = np.random.default_rng(B + S)
    lens = rng.integers(1, min(S, 700) + 1, size=B)
    lens[0] = S
    lens[1:3] = (0, 1)[:max(0, min(2, B - 1))]
    width = -(-S // 64)
    pages = int(sum(-(-n // 64) for n in lens)) + 1
    c = Cache(cuda, rng, dtype, pages, 64, H)
    table, at = np.zeros((B, width), np.int32), rng.permutation(pages)
    for b, n in enumerate(lens):
        table[b, :-(-n // 64)], at = at[:-(-n // 64)], at[-(-n // 64):]
    q = _x(rng, B, 3 * H, 128)
    _decode(cuda, c, q, table, lens.tolist(), what, max_seqlen=S)


def test_decode_least_workspace(cuda):
    """A caller's workspace that holds 4096-token splits only, one that holds the
    even sharing, and one too small."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(83)
    c = Cache(cuda, rng, "e4m3", 300, 64, 4)
    table, lens = _for_teams(cuda, _table(rng, 2, 150, 300), 64, 4), [9500, 4097]
    q = _x(rng, 2, 16, 128)
    n = -(-table.shape[1] * 64 // 4096)
    least = -(-2 * 16 * n * 512 // 256) * 256 + -(-2 * 16 * n * 8 // 256) * 256 + 4 * (1 + 2 * n)
    for size in (least, 64 << 20):
        ws = torch.empty(size, dtype=torch.uint8, device=cuda)
        _decode(cuda, c, q, table, lens, f"workspace {size}", workspace=ws)
    with pytest.raises(fg.FgqaError):
        fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens), workspace=ws[:least - 4],
                                  **c.scales)


@pytest.mark.parametrize("what", ["append", "decode", "weights", "evict"])
def test_offsets_past_32_bits(cuda, what):
    """Pages that begin past 4 GiB of a cache."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(90)
    P, H = 64, 8
    pages = (1 << 32) // (P * H * 128) + 12
    small = Cache(cuda, rng, "e4m3", 12, P, H)
    big, s = [], []
    for i in range(2):
        t = torch.empty((pages, P, H, 128), dtype=torch.uint8, device=cuda)
        t[-12:] = small.t[i].view(torch.uint8)
        big.append(t.view(torch.float8_e4m3fn))
        f = torch.ones((pages, H), dtype=torch.float32, device=cuda)
        f[-12:] = small.s[i]
        s.append(f)
    near, lens, B = _table(rng, 2, 3, 6), [150, 100], 2
    far = near + (pages - 12)
    q = _x(rng, B, 16, 128).to(cuda)
    res = []
    for t, sc, table, off in ((small.t, small.s, near, 0), (big, s, far, pages - 12)):
        kw = dict(k_scale=sc[0], v_scale=sc[1])
        tb, ln = _i32(cuda, table), _i32(cuda, lens)
        if what == "append":
            x = _x(np.random.default_rng(91), B, 30, H, 128).to(cuda)
            fg.append_kv_paged(x, x, t[0], t[1], tb, ln, **kw)
            out = ()
        elif what == "decode":
            out = (fg.decode_flash_gqa_paged(q, t[0], t[1], tb, ln, **kw),)
        elif what == "weights":
            lse = torch.full((B, 16), 5.0, device=cuda)
            out = (fg.accumulate_kv_weights_paged(q, t[0], lse, tb, ln, torch.zeros((B, H, 192), device=cuda),
                                                  k_scale=sc[0]),)
        else:
            w = torch.rand((B, H, 192), device=cuda, generator=torch.Generator(cuda).manual_seed(1))
            new = _i32(cuda, np.array([[6, 7], [8, 9]]) + off)
            out = fg.evict_kv_paged(t[0], t[1], tb, ln, w, new, budget=80, recent=8, **kw)
        torch.cuda.synchronize()
        tail = [x[-12:].view(torch.uint8) for x in t] + [x[-12:] for x in sc]
        res.append([x.clone() for x in (*out, *tail)])
    for a, b in zip(*res):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ weights
def _weights(cuda, c, q, table, lens, lse, w, what, **kw):
    torch = _torch()
    scales = {k: v for k, v in c.scales.items() if k == "k_scale"}
    start = w.cpu().double().numpy().copy()
    got = _fg().accumulate_kv_weights_paged(q.to(cuda), c.t[0], lse, _i32(cuda, table), _i32(cuda, lens), w, **scales, **kw)
    torch.cuda.synchronize()
    assert got is w
    add, tol = ref.weights(q.float().numpy().astype(np.float64), c.n[0], c.sn[0], table, lens, lse.cpu().double().numpy(),
                           SCALE, w.shape[2], whole=0.25 if c.dtype == "e4m3" else 1.0)
    got = got.cpu().double().numpy()
    # (a made-up LSE can lie far below the scores: sums past fp32's largest number are inf)
    with np.errstate(over="ignore", invalid="ignore"):
        want = start + add
        over = want > float(np.finfo(np.float32).max)
        bad = np.where(over, ~np.isposinf(got), ~(np.abs(got - want) <= tol + 2.0 ** -23 * np.abs(want)))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, first at {np.argwhere(bad)[0].tolist()}: " \
                          f"{got[bad][0]} for {want[bad][0]}"
    for b, n in enumerate(lens):
        assert np.array_equal(got[b, :, n:], start[b, :, n:]), f"{what}: weights past the length"


@pytest.mark.parametrize("dtype,scales", KINDS)
@pytest.mark.parametrize("P", [1, 4, 8, 16, 32, 64, 256])
def test_weights_page_sizes(cuda, P, dtype, scales):
    torch = _torch()
    what = f"weights P={P} {dtype} scales={scales}"
    print(what, flush=True)
    rng = np.random.default_rng(100 + P)
    lens = [700, 1, 333, 0, 32, 65]
    width = -(-700 // P)
    c = Cache(cuda, rng, dtype, len(lens) * width + 2, P, 2, scales=scales)
    table = _table(rng, len(lens), width, len(lens) * width + 2)
    q = _x(rng, len(lens), 10, 128)
    lse = torch.from_numpy(rng.uniform(3, 12, size=(len(lens), 10)).astype(np.float32)).to(cuda)
    w = torch.from_numpy(rng.uniform(0, 1, size=(len(lens), 2, 711)).astype(np.float32)).to(cuda)
    _weights(cuda, c, q, table, lens, lse, w, what, max_seqlen=700)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("G,H", [(1, 1), (4, 3), (7, 4), (16, 2), (1, 8)])
def test_weights_heads(cuda, G, H, dtype):
    torch = _torch()
    rng = np.random.default_rng(120 + G)
    lens = [97, 260]
    c = Cache(cuda, rng, dtype, 40, 16, H, pad=1)
    table = _table(rng, 2, 17, 40)
    wide = torch.from_numpy(rng.uniform(0, 1, size=(2, H + 1, 300)).astype(np.float32)).to(cuda)
    lse = torch.from_numpy(rng.uniform(3, 12, size=(2, G * H)).astype(np.float32)).to(cuda)
    _weights(cuda, c, _x(rng, 2, G * H, 128), table, lens, lse, wide[:, 1:, 3:], f"heads {G} {H} {dtype}")


@pytest.mark.parametrize("dtype,P", [("int8", 8), ("bf16", 4), ("e4m3", 64)])
def test_weights_several_items_a_wave(cuda, dtype, P):
    """More items than waves: a sequence's waves take items in turn, up to its length."""
    torch = _torch()
    rng = np.random.default_rng(130)
    B, W = 1024, 4500   # 64 waves a row: 4096 tokens
    lens = rng.integers(0, 4, size=B)
    lens[[3, 500, 1023]] = (4500, 4096, 4161)
    width = -(-W // P)
    need = [-(-int(n) // P) for n in lens]
    pages = sum(need) + 1
    c = Cache(cuda, rng, dtype, pages, P, 2, scales=dtype != "bf16")
    table, at = np.full((B, width), -1, np.int32), rng.permutation(pages)
    for b, n in enumerate(need):
        table[b, :n], at = at[:n], at[n:]
    q = _x(rng, B, 4, 128)
    lse = torch.from_numpy(rng.uniform(3, 12, size=(B, 4)).astype(np.float32)).to(cuda)
    w = torch.from_numpy(rng.uniform(0, 1, size=(B, 2, W)).astype(np.float32)).to(cuda)
    _weights(cuda, c, q, table, lens.tolist(), lse, w, f"several items {dtype} P={P}", max_seqlen=W)


def test_weights_sum_to_the_query_heads(cuda):
    """With the decode's LSE the weights of a step are a softmax's: they add up to
    G; a long sequence and one of a single token."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(130)
    c = Cache(cuda, rng, "int8", 160, 64, 2)
    table, lens = _table(rng, 2, 80, 160), [5000, 1]
    q = _x(rng, 2, 14, 128)
    lse = torch.empty((2, 14), device=cuda)
    fg.decode_flash_gqa_paged(q.to(cuda), c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens), lse=lse, **c.scales)
    w = torch.zeros((2, 2, 5120), device=cuda)
    _weights(cuda, c, q, table, lens, lse, w, "with the decode's lse")
    total = w.double().sum(dim=2).cpu().numpy()
    o, l, m, err = ref.decode(q.float().numpy().astype(np.float64), c.n[0], c.sn[0], c.n[1], c.sn[1], table, lens, SCALE)
    assert np.all(np.abs(total - 7) <= 7 * (2.1 * err.max() + 2.0 ** -24 * 10100 + 2.0 ** -21 * np.abs(l).max()))


def test_weights_same_bits_every_time(cuda):
    torch = _torch()
    rng = np.random.default_rng(131)
    c = Cache(cuda, rng, "e4m3", 100, 16, 2)
    table, lens = _i32(cuda, _table(rng, 2, 50, 100)), _i32(cuda, [777, 800])
    q = _x(rng, 2, 16, 128).to(cuda)
    lse = torch.full((2, 16), 7.0, device=cuda)
    runs = [_fg().accumulate_kv_weights_paged(q, c.t[0], lse, table, lens, torch.zeros((2, 2, 800), device=cuda),
                                              k_scale=c.s[0]) for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


# ------------------------------------------------------------------ evict
def _evict(cuda, c, table, new_table, lens, w, budget, recent, what, **kw):
    torch = _torch()
    start = w.cpu().clone()
    nl, nw, kept = _fg().evict_kv_paged(c.t[0], c.t[1], _i32(cuda, table), _i32(cuda, lens), w, _i32(cuda, new_table),
                                        budget=budget, recent=recent, **c.scales, **kw)
    torch.cuda.synchronize()
    assert torch.equal(w.cpu().view(torch.int32), start.view(torch.int32)), f"{what}: the input weights changed"
    rl, rw, rk = ref.evict(c.n[0], c.sn[0], c.n[1], c.sn[1], c.dtype, table, new_table, np.array(lens),
                           start.numpy(), budget, recent)
    assert np.array_equal(kept.cpu().numpy(), rk), f"{what}: kept"
    assert np.array_equal(nl.cpu().numpy(), rl), f"{what}: lengths"
    assert np.array_equal(nw.cpu().numpy(), rw, equal_nan=True), f"{what}: weights"
    c.check(what)
    return nl, nw, kept


@pytest.mark.parametrize("dtype,scales", KINDS)
@pytest.mark.parametrize("P", [1, 4, 8, 16, 64, 128, 512])
def test_evict_page_sizes(cuda, P, dtype, scales):
    torch = _torch()
    what = f"evict P={P} {dtype} scales={scales}"
    print(what, flush=True)
    rng = np.random.default_rng(200 + P)
    lens = [600, 0, 1, 99, 100, 101, 333]
    width, nwidth = -(-600 // P), -(-100 // P)
    pages = len(lens) * (width + nwidth)
    c = Cache(cuda, rng, dtype, pages, P, 2, scales=scales)
    both = _table(rng, len(lens), width + nwidth, pages)
    w = torch.from_numpy(rng.exponential(size=(len(lens), 2, 600)).astype(np.float32)).to(cuda)
    _evict(cuda, c, both[:, :width], both[:, width:], lens, w, 100, 17, what)


@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (64, 200), (299, 0), (300, 5), (1000, 10)])
def test_evict_budgets(cuda, budget, recent):
    torch = _torch()
    rng = np.random.default_rng(220)
    lens = [300, 65, 64, 2]
    nwidth = -(-min(budget, 320) // 16)
    pages = 4 * (20 + nwidth)
    c = Cache(cuda, rng, "int8", pages, 16, 1)
    both = _table(rng, 4, 20 + nwidth, pages)
    w = torch.from_numpy(rng.exponential(size=(4, 1, 320)).astype(np.float32)).to(cuda)
    _evict(cuda, c, both[:, :20], both[:, 20:], lens, w, budget, recent, f"budget {budget} recent {recent}")


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "special", "negative", "close", "sorted", "falling"])
def test_evict_weights_of_every_kind(cuda, kind):
    """Ties (all equal, few values, signed zeros), infinities, NaN, negative and
    subnormal weights, weights that differ in the last bit only, ordered rows."""
    torch = _torch()
    rng = np.random.default_rng(230)
    n = 2500
    w = {"equal": lambda: np.full((1, 2, n), 0.25),
         "few": lambda: rng.integers(0, 3, size=(1, 2, n)) * 0.5,
         "zeros": lambda: np.where(rng.integers(0, 2, size=(1, 2, n)) == 1, 0.0, -0.0),
         "special": lambda: rng.choice([np.inf, -np.inf, np.nan, -np.nan, 0.0, -0.0, 1.0, 1e-45, -1e-45, 3e38], size=(1, 2, n)),
         "negative": lambda: rng.standard_normal((1, 2, n)),
         "close": lambda: (0x3f000000 + rng.integers(0, 40, size=(1, 2, n))).astype(np.uint32).view(np.float32),
         "sorted": lambda: np.sort(rng.exponential(size=(1, 2, n))),
         "falling": lambda: -np.sort(-rng.exponential(size=(1, 2, n)))}[kind]().astype(np.float32)
    width, budget = -(-n // 32), 1111
    nwidth = -(-budget // 32)
    c = Cache(cuda, rng, "e4m3", width + nwidth, 32, 2)
    both = _table(rng, 1, width + nwidth, width + nwidth)
    _evict(cuda, c, both[:, :width], both[:, width:], [n], torch.from_numpy(w).to(cuda), budget, 100, kind)


def test_evict_long_row(cuda):
    """More tokens than any single pass of the selection holds; strided weights and outputs given."""
    torch = _torch()
    rng = np.random.default_rng(240)
    n, budget, P = 70001, 5003, 256
    width, nwidth = -(-n // P), -(-budget // P)
    c = Cache(cuda, rng, "bf16", width + nwidth, P, 1)
    both = _table(rng, 1, width + nwidth, width + nwidth)
    wide = torch.from_numpy(rng.exponential(size=(1, 3, n + 5)).astype(np.float32)).to(cuda)
    out = torch.full((1, 1, n + 2), -1.0, device=cuda)
    kept = torch.empty((1, 1, budget), dtype=torch.int32, device=cuda)
    lens = torch.empty((1,), dtype=torch.int32, device=cuda)
    got = _evict(cuda, c, both[:, :width], both[:, width:], [n], wide[:, 1:2, 3:], budget, 1000, "long row",
                 new_weights=out, kept=kept, new_seqlens=lens, max_seqlen=n)
    assert got[0] is lens and got[1] is out and got[2] is kept


@pytest.mark.parametrize("n", [8192, 8193, 20000, 32768, 32769])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_few_rows(cuda, n, ties):
    """Rows that several workgroups share, at the ends of what one holds, beside a
    short sequence, one of candidates 1 past a multiple of 4 and one that is cut to its recent tokens."""
    torch = _torch()
    rng = np.random.default_rng(n)
    lens = [n, 5 + 128, n - 2, 129]
    budget, recent, P = 1999, 128, 512
    width, nwidth = -(-n // P), -(-budget // P)
    pages = 4 * (width + nwidth)
    c = Cache(cuda, rng, "int8", pages, P, 1)
    both = _table(rng, 4, width + nwidth, pages)
    w = rng.integers(0, 9, size=(4, 1, n)) if ties else rng.exponential(size=(4, 1, n))
    _evict(cuda, c, both[:, :width], both[:, width:], lens, torch.from_numpy(w.astype(np.float32)).to(cuda), budget, recent,
           f"few rows n={n} ties={ties}")
    w = torch.from_numpy(w[:, :, :n].astype(np.float32)).to(cuda)
    for budget in (1, 130, n - 3):   # the candidates' last vector of 4 in every place
        if -(-budget // P) <= nwidth:
            _evict(cuda, c, both[:, :width], both[:, width:], lens, w, budget, min(budget, recent), f"n={n} budget={budget}")


@pytest.mark.parametrize("cand", [1, 2, 3, 4, 5, 6, 7, 63, 257, 4095, 4097])
def test_evict_candidates_past_the_last_vector(cuda, cand):
    """Candidates in every place of the last 4; what lies behind them is larger."""
    torch = _torch()
    rng = np.random.default_rng(cand)
    recent, P = 3, 64
    n = cand + recent
    budget = recent + max(1, cand // 2)
    if budget >= n:
        n, recent, budget = cand + 1, 1, 1
    width, nwidth = -(-n // P), -(-budget // P)
    c = Cache(cuda, rng, "e4m3", width + nwidth, P, 1)
    both = _table(rng, 1, width + nwidth, width + nwidth)
    w = rng.exponential(size=(1, 1, n + 5)).astype(np.float32)
    w[:, :, n - recent:] = 1e30
    _evict(cuda, c, both[:, :width], both[:, width:], [n], torch.from_numpy(w).to(cuda), budget, recent, f"candidates {cand}")


def test_evict_pages_outside(cuda):
    """New pages outside the cache are not written; old entries are clamped."""
    torch = _torch()
    rng = np.random.default_rng(250)
    c = Cache(cuda, rng, "int8", 30, 16, 2, pad=2)
    both = _table(rng, 2, 12, 30)
    table, new = both[:, :8].copy(), both[:, 8:].copy()
    new[0, 1], new[1, 0] = -1, 30
    w = torch.from_numpy(rng.exponential(size=(2, 2, 128)).astype(np.float32)).to(cuda)
    _evict(cuda, c, table, new, [128, 120], w, 60, 8, "pages outside")


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype,P", [("e4m3", 16), ("int8", 64), ("int8", 8)])
def test_a_conversation(cuda, dtype, P):
    """Prompts, steps, an eviction and steps after it, each checked: what a server does."""
    torch = _torch()
    rng = np.random.default_rng(300 + P)
    B, H, G, budget = 3, 2, 4, 90
    width, nwidth = -(-200 // P), -(-120 // P)
    pages = B * (width + nwidth)
    c = Cache(cuda, rng, dtype, pages, P, H)
    both = _table(rng, B, width + nwidth, pages)
    table, lens = both[:, :width], np.array([0, 0, 0])
    news = np.array([150, 33, 90])
    _append(cuda, c, _x(rng, B, 150, H, 128), _x(rng, B, 150, H, 128), table, lens, news, "prompt")
    lens = lens + news
    w = torch.zeros((B, H, 200), device=cuda)
    for step in range(6):
        _append(cuda, c, _x(rng, B, 1, H, 128), _x(rng, B, 1, H, 128), table, lens, None, f"step {step}")
        lens = lens + 1
        q = _x(rng, B, G * H, 128)
        _, lse = _decode(cuda, c, q, table, lens.tolist(), f"step {step}")
        _weights(cuda, c, q, table, lens.tolist(), lse, w, f"step {step}")
        if step == 2:
            nl, w, _ = _evict(cuda, c, table, both[:, width:], lens.tolist(), w, budget, 10, "evict")
            lens, table = nl.cpu().numpy().astype(np.int64), both[:, width:]


def test_graph_of_a_step_replayed(cuda):
    """Append, decode and weights of a step captured once; the lengths advance on
    the device between replays, with eager work in between; each replay gives
    what the eager calls give on a copy."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(310)
    B, H, Hq, P = 2, 2, 8, 16
    c = Cache(cuda, rng, "int8", 30, P, H)
    table = _i32(cuda, _table(rng, B, 15, 30))

    def state():
        return dict(k=c.t[0].clone(), v=c.t[1].clone(), ks=c.s[0].clone(), vs=c.s[1].clone(),
                    lens=_i32(cuda, [30, 100]), w=torch.zeros((B, H, 240), device=cuda),
                    x=torch.zeros((B, 1, H, 128), dtype=torch.bfloat16, device=cuda),
                    q=torch.zeros((B, Hq, 128), dtype=torch.bfloat16, device=cuda),
                    lse=torch.empty((B, Hq), device=cuda))

    def step(s):
        fg.append_kv_paged(s["x"], s["x"], s["k"], s["v"], table, s["lens"], k_scale=s["ks"], v_scale=s["vs"])
        s["lens"] += 1
        s["o"] = fg.decode_flash_gqa_paged(s["q"], s["k"], s["v"], table, s["lens"], k_scale=s["ks"], v_scale=s["vs"],
                                           lse=s["lse"])
        fg.accumulate_kv_weights_paged(s["q"], s["k"], s["lse"], table, s["lens"], s["w"], k_scale=s["ks"])

    a, b = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)      # warm-up on the copy's twin, undone below
    torch.cuda.current_stream().wait_stream(side)
    a = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for i in range(5):
        x, q = _x(rng, B, 1, H, 128).to(cuda) * 2.0 ** i, _x(rng, B, Hq, 128).to(cuda)
        for s in (a, b):
            s["x"].copy_(x)
            s["q"].copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        step(b)
        torch.cuda.synchronize()
        for name in ("lens", "ks", "vs", "lse", "w"):
            assert torch.equal(a[name], b[name]), f"replay {i}: {name}"
        for name in ("k", "v", "o"):
            assert torch.equal(a[name].view(torch.uint8), b[name].view(torch.uint8)), f"replay {i}: {name}"


def test_two_streams_at_once(cuda):
    """Decodes, without workspaces of their own given, and evictions on two
    streams at the same time give what they give alone."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(320)
    c = Cache(cuda, rng, "e4m3", 400, 16, 4)
    both = _table(rng, 4, 100, 400)
    qs = [_x(rng, 2, 32, 128).to(cuda) for _ in range(2)]
    w = torch.from_numpy(rng.exponential(size=(2, 4, 1280)).astype(np.float32)).to(cuda)
    args = [(_i32(cuda, both[2 * i:2 * i + 2, :80]), _i32(cuda, [1280 - 100 * i, 700]),
             _i32(cuda, both[2 * i:2 * i + 2, 80:])) for i in range(2)]

    def work(i):
        table, lens, new = args[i]
        o = fg.decode_flash_gqa_paged(qs[i], c.t[0], c.t[1], table, lens, **c.scales)
        return (o,) + fg.evict_kv_paged(c.t[0], c.t[1], table, lens, w, new, budget=300, recent=20, **c.scales)

    alone = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


@pytest.mark.parametrize("teams", [False, True])
def test_two_graphs_at_once(cuda, teams):
    """Two captured decodes (in splits or over teams, merged through a workspace) and
    evictions (a row shared by several workgroups), replayed on two streams at once
    with eager work between the replays."""
    torch = _torch()
    fg = _fg()
    rng = np.random.default_rng(330)
    P, n = 64, 9000
    c = Cache(cuda, rng, "int8", 2 * 180, P, 4)
    both = _table(rng, 2, 180, 360)
    tables = [_for_teams(cuda, both[i:i + 1, :141], P, 4) if teams else both[i:i + 1, :141] for i in range(2)]
    args = [(_x(rng, 1, 16, 128).to(cuda), _i32(cuda, tables[i]), _i32(cuda, [n - 77 * i]), _i32(cuda, both[i:i + 1, 141:]))
            for i in range(2)]
    w = torch.from_numpy(rng.exponential(size=(2, 4, n)).astype(np.float32)).to(cuda)

    def work(i):
        q, table, lens, new = args[i]
        o = fg.decode_flash_gqa_paged(q, c.t[0], c.t[1], table, lens, **c.scales)
        return (o,) + fg.evict_kv_paged(c.t[0], c.t[1], table, lens, w[i:i + 1], new, budget=2000, recent=100,
                                        max_seqlen=n, **c.scales)

    alone = [work(0), work(1)]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            outs.append(work(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(6):
        for got in outs:
            for x in got:
                x.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(alone, outs):
            for x, y in zip(a, b):
                assert torch.equal(x, y), f"replay {r}"
        for a, b in zip(alone, [work(0), work(1)]):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


# ------------------------------------------------------------------ C++ operator layer
def test_cplusplus_entry_points(cuda):
    """The C++ entry points on the default stream against the Python functions: the same bits."""
    import ctypes
    import subprocess

    import cuda_llm_ops_amd._lib as L
    torch = _torch()
    fg = _fg()

    class Kv(ctypes.Structure):   # KvCache (kv_cache_kernel.h)
        _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("ks", ctypes.c_void_p), ("vs", ctypes.c_void_p),
                    ("type", ctypes.c_int), ("pages", ctypes.c_int), ("page", ctypes.c_int), ("heads", ctypes.c_int),
                    ("k_scale", ctypes.c_float), ("v_scale", ctypes.c_float)]

    syms = subprocess.run(["nm", "-D", "--defined-only", L.LIB_PATH], check=True, capture_output=True, text=True).stdout
    lib = L.lib()

    def entry(name):
        return getattr(lib, next(w.split()[-1] for w in syms.splitlines() if f"{len(name)}{name}R" in w))

    status = getattr(lib, next(w.split()[-1] for w in syms.splitlines() if "FlashGqaGetLastStatus" in w))
    rng = np.random.default_rng(400)
    B, H, Hq, P, pages = 2, 2, 8, 16, 30
    c = Cache(cuda, rng, "int8", pages, P, H)
    table = _i32(cuda, _table(rng, B, 10, 20))
    new_table = _i32(cuda, 20 + np.arange(10).reshape(2, 5))
    lens, news = _i32(cuda, [100, 37]), _i32(cuda, [5, 3])
    x = _x(rng, B, 5, H, 128).to(cuda)
    q = _x(rng, B, Hq, 128).to(cuda)
    P_ = lambda t: ctypes.c_void_p(0 if t is None else t.data_ptr())  # noqa: E731
    f32, i32 = ctypes.c_float, ctypes.c_int
    results = []
    for cpp in (False, True):
        k, v, ks, vs = c.t[0].clone(), c.t[1].clone(), c.s[0].clone(), c.s[1].clone()
        o = torch.empty((B, Hq, 128), dtype=torch.bfloat16, device=cuda)
        lse, w = torch.empty((B, Hq), device=cuda), torch.zeros((B, H, 10 * P), device=cuda)
        nw, kept, nl = torch.empty_like(w), torch.empty((B, H, 70), dtype=torch.int32, device=cuda), torch.empty_like(lens)
        torch.cuda.synchronize()
        after = lens + news
        if cpp:
            torch.cuda.synchronize()
            kv = Kv(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), 2, pages, P, H, 1.0, 1.0)
            ref_kv = ctypes.byref(kv)
            entry("LaunchKvCacheAppendKernel")(ref_kv, P_(x), P_(x), P_(table), P_(lens), P_(news), i32(B), i32(5), i32(10))
            assert status() == 0
            entry("LaunchFlashGqaBf16KernelPagedBlocks")(ref_kv, P_(q), f32(SCALE), P_(o), P_(lse), P_(table), P_(after),
                                                         i32(B), i32(10), i32(Hq))
            assert status() == 0
            entry("LaunchKvCacheWeightsKernel")(ref_kv, P_(q), f32(SCALE), P_(lse), P_(w), P_(table), P_(after), i32(B),
                                                i32(10), i32(Hq))
            assert status() == 0
            entry("LaunchKvCacheEvictKernel")(ref_kv, P_(w), P_(nw), P_(table), P_(new_table), P_(after), P_(nl), P_(kept),
                                              i32(70), i32(8), i32(B), i32(10), i32(5))
            assert status() == 0
            entry("LaunchKvCacheEvictKernel")(ref_kv, P_(w), P_(nw), P_(table), P_(new_table), P_(after), P_(nl), P_(kept),
                                              i32(0), i32(8), i32(B), i32(10), i32(5))
            assert status() == L.FGQA_ERR_INVALID_ARGUMENT
        else:
            sc = dict(k_scale=ks, v_scale=vs)
            fg.append_kv_paged(x, x, k, v, table, lens, new_lens=news, **sc)
            fg.decode_flash_gqa_paged(q, k, v, table, after, out=o, lse=lse, **sc)
            fg.accumulate_kv_weights_paged(q, k, lse, table, after, w, k_scale=ks)
            fg.evict_kv_paged(k, v, table, after, w, new_table, 70, 8, new_seqlens=nl, new_weights=nw, kept=kept, **sc)
        torch.cuda.synchronize()
        results.append([t.clone() for t in (k, v, ks, vs, o.view(torch.int16), lse, w, nw, kept, nl)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
