"""The C++ entry points of qk_norm_rope_kernel.h and kv_pages_kernel.h, on the default stream,
against the Python functions: the same bits."""
import ctypes
import random
import subprocess
from ctypes import c_bool, c_float, c_int, c_void_p

import pytest

pytestmark = pytest.mark.gpu


class Kv(ctypes.Structure):   # KvCache (kv_cache_kernel.h)
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("ks", c_void_p), ("vs", c_void_p), ("type", c_int), ("pages", c_int),
                ("page", c_int), ("heads", c_int), ("k_scale", c_float), ("v_scale", c_float)]


class QkNormRope(ctypes.Structure):   # qk_norm_rope_kernel.h
    _fields_ = [("positions", c_void_p), ("inv_freq", c_void_p), ("axes", c_void_p), ("q_weight", c_void_p), ("k_weight", c_void_p),
                ("eps", c_float), ("num_axes", c_int), ("batch", c_int), ("seqlen", c_int), ("hq", c_int), ("hkv", c_int),
                ("head_dim", c_int), ("rotary_dim", c_int), ("interleaved", c_bool)]


@pytest.fixture(scope="module")
def entries():
    """(entry point by name, the status of the last call)."""
    import cuda_llm_ops_amd._lib as L
    syms = subprocess.run(["nm", "-D", "--defined-only", L.LIB_PATH], check=True, capture_output=True, text=True).stdout
    lib = L.lib()

    def entry(name):
        return getattr(lib, next(w.split()[-1] for w in syms.splitlines() if f"{len(name)}{name}R" in w))

    return entry, getattr(lib, next(w.split()[-1] for w in syms.splitlines() if "FlashGqaGetLastStatus" in w))


def _p(t):
    return c_void_p(0 if t is None else t.data_ptr())


@pytest.mark.parametrize("norm", (False, True))
def test_norm_and_rotation(cuda, entries, norm):
    import torch
    import cuda_llm_ops_amd as fg
    import cuda_llm_ops_amd._lib as L
    entry, status = entries
    g = torch.Generator(device=cuda).manual_seed(3)
    B, S, Hq, Hkv, D, R = 2, 37, 6, 2, 96, 64
    q, gq = (torch.randn(B, S, Hq, D, generator=g, device=cuda).bfloat16() for _ in range(2))
    k, gk = (torch.randn(B, S, Hkv, D, generator=g, device=cuda).bfloat16() for _ in range(2))
    pos = torch.randint(0, 500, (3, B, S), generator=g, device=cuda, dtype=torch.int32)
    inv_freq = torch.rand(R // 2, generator=g, device=cuda)
    axes = torch.randint(0, 3, (R // 2,), generator=g, device=cuda, dtype=torch.int32)
    w = [(1 + 0.1 * torch.randn(D, generator=g, device=cuda)).bfloat16() for _ in range(2)] if norm else [None, None]
    kw = dict(axes=axes, interleaved=True, eps=1e-5)
    if norm:
        kw.update(q_weight=w[0], k_weight=w[1])
    want = [*fg.qk_norm_rope(q, k, pos, inv_freq, **kw),
            *(t for t in fg.qk_norm_rope_backward(gq, gk, *((q, k) if norm else (None, None)), pos, inv_freq, **kw) if t is not None)]
    how = QkNormRope(pos.data_ptr(), inv_freq.data_ptr(), axes.data_ptr(), _p(w[0]), _p(w[1]), 1e-5, 3, B, S, Hq, Hkv, D, R, True)
    qo, ko, dq, dk = (torch.zeros_like(t) for t in (q, k, q, k))
    dw = [torch.zeros(D, device=cuda) for _ in range(2)] if norm else [None, None]
    torch.cuda.synchronize()
    entry("LaunchQkNormRopeBf16Kernel")(ctypes.byref(how), _p(q), _p(k), _p(qo), _p(ko))
    assert status() == 0
    entry("LaunchQkNormRopeBackwardBf16Kernel")(ctypes.byref(how), _p(q if norm else None), _p(k if norm else None), _p(gq), _p(gk),
                                                _p(dq), _p(dk), _p(dw[0]), _p(dw[1]))
    assert status() == 0
    torch.cuda.synchronize()
    out = [qo, ko, dq, dk] + (dw if norm else [])
    assert len(out) == len(want)
    for a, b in zip(out, want):
        assert torch.equal(a, b)
    how.rotary_dim = D + 16
    entry("LaunchQkNormRopeBf16Kernel")(ctypes.byref(how), _p(q), _p(k), _p(qo), _p(ko))
    assert status() == L.FGQA_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", ("bf16", "e4m3", "int8"))
def test_pages(cuda, entries, dtype):
    """Fork, a decode of what is then shared, and compact."""
    import torch
    import cuda_llm_ops_amd as fg
    import cuda_llm_ops_amd._lib as L
    entry, status = entries
    r = random.Random(8)
    g = torch.Generator(device=cuda).manual_seed(5)
    B, N, P, H, Hq, W, pages = 2, 6, 16, 2, 8, 30, 90
    kind = {"bf16": 0, "e4m3": 1, "int8": 2}[dtype]
    if dtype == "int8":
        data = [torch.randint(-128, 128, (pages, P, H, 128), generator=g, device=cuda, dtype=torch.int8) for _ in range(2)]
    else:
        data = [torch.randn(pages, P, H, 128, generator=g, device=cuda).to(torch.bfloat16 if kind == 0 else torch.float8_e4m3fn)
                for _ in range(2)]
    scales = [] if kind == 0 else [0.01 + 0.01 * torch.rand(pages, H, generator=g, device=cuda) for _ in range(2)]
    order = list(range(pages))
    r.shuffle(order)
    lens = [300, 41]
    i32 = dict(dtype=torch.int32, device=cuda)
    table = torch.tensor([[order.pop() if j * P < n else -1 for j in range(W)] for n in lens], **i32)
    lens_t, parents, new = torch.tensor(lens, **i32), torch.tensor([0, 0, 1, 0, -1, 0], **i32), torch.tensor([3] * N, **i32)
    starts, shared = torch.tensor([0, 2], **i32), torch.tensor([288], **i32)
    q = torch.randn(N, Hq, 128, generator=g, device=cuda).bfloat16()
    results = []
    for cpp in (False, True):
        k, v = (t.clone() for t in data)
        s = [t.clone() for t in scales]
        t1, t2 = torch.full((N, W), -9, **i32), torch.full((N, W), -9, **i32)
        n1, free, used = torch.full((N,), -9, **i32), torch.full((1,), -9, **i32), torch.full((1,), -9, **i32)
        o, lse = torch.zeros(N, Hq, 128, dtype=torch.bfloat16, device=cuda), torch.zeros(N, Hq, device=cuda)
        torch.cuda.synchronize()
        if cpp:
            ks, vs = (_p(t) for t in s) if s else (c_void_p(0), c_void_p(0))
            kv = Kv(k.data_ptr(), v.data_ptr(), ks, vs, kind, pages, P, H, 1.0, 1.0)
            cache = ctypes.byref(kv)
            entry("LaunchKvCacheForkKernel")(cache, _p(table), _p(lens_t), _p(parents), _p(new), c_void_p(0), _p(t1), _p(n1),
                                             _p(free), c_int(B), c_int(W), c_int(N), c_int(W))
            assert status() == 0
            entry("LaunchFlashGqaBf16KernelPagedShared")(cache, _p(q), c_float(0.0625), _p(o), _p(lse), _p(t1), _p(n1), _p(starts),
                                                         _p(shared), c_int(N), c_int(W), c_int(Hq), c_int(1))
            assert status() == 0
            entry("LaunchKvCacheCompactKernel")(cache, _p(t1), _p(n1), c_void_p(0), _p(t2), _p(used), c_int(N), c_int(W))
            assert status() == 0
            entry("LaunchKvCacheCompactKernel")(cache, _p(t1), _p(n1), c_void_p(0), _p(t2), c_void_p(0), c_int(N), c_int(W))
            assert status() == L.FGQA_ERR_INVALID_ARGUMENT
        else:
            sc = dict(zip(("k_scale", "v_scale"), s))
            fg.fork_kv_paged(k, v, table, lens_t, parents=parents, new_lens=new, new_block_table=t1, new_seqlens=n1, num_free=free, **sc)
            fg.decode_flash_gqa_paged_shared(q, k, v, t1, n1, starts, shared, scale=0.0625, out=o, lse=lse, **sc)
            fg.compact_kv_paged(k, v, t1, n1, new_block_table=t2, num_used=used, **sc)
        torch.cuda.synchronize()
        results.append([t.contiguous().view(-1).view(torch.uint8).clone() for t in (k, v, *s, t1, t2, n1, free, used, o, lse)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert bool((results[0][-1] != 0).any())
