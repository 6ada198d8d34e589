"""CPU tests of the paged KV cache's operators: the host validation and the C++
operator layer under sanitizers, the Python binding's layout against the header,
exported entry points, and every refusal of the Python functions (all before any
GPU is looked at)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import cuda_llm_ops_amd as fg
from cuda_llm_ops_amd import _lib, flash_gqa, kv_cache
from tests.test_host_sanitizers import HOST, ROOT, _build_and_run

HEADER = os.path.join(ROOT, "include", "fgqa_kv.h")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_kv_plan_and_operator_layer_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_kv_plan",
                   [os.path.join(HOST, "fgqa_plan.cpp"), os.path.join(HOST, "kv_plan.cpp"),
                    os.path.join(ROOT, "src", "cplusplus", "FlashGQA", "kv_cache.cpp"),
                    os.path.join(ROOT, "tests", "host", "test_kv_plan.cpp")])


def test_exported():
    names = set(re.findall(r"^int (fgqa_\w+)\(", open(HEADER).read(), flags=re.M))
    assert names == {"fgqa_kv_append", "fgqa_decode_blocks", "fgqa_decode_blocks_workspace_bytes", "fgqa_kv_weights",
                     "fgqa_kv_evict"}
    syms = subprocess.run(["nm", "-D", "--defined-only", "-C", _lib.LIB_PATH], check=True, capture_output=True,
                          text=True).stdout
    for n in names:
        assert re.search(rf"\bT {n}$", syms, flags=re.M), n
    hdr = open(os.path.join(ROOT, "include", "cplusplus", "FlashGQA", "kv_cache_kernel.h")).read()
    for d in re.findall(r"^void (\w+)\(", hdr, flags=re.M):
        assert re.search(rf"\bT {d}\(", syms), d


# ------------------------------------------------------------------ refusals
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _append(**kw):
    a = dict(k=torch.zeros(2, 3, 4, 128, dtype=BF), v=torch.zeros(2, 3, 4, 128, dtype=BF),
             k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             block_table=torch.zeros(2, 5, dtype=torch.int32), seqlens=torch.zeros(2, dtype=torch.int32),
             k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.append_kv_paged(**a)


def _decode(**kw):
    a = dict(q=torch.zeros(2, 8, 128, dtype=BF), k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), block_table=torch.zeros(2, 5, dtype=torch.int32),
             seqlens=torch.zeros(2, dtype=torch.int32), k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.decode_flash_gqa_paged(**a)


def _weights(**kw):
    a = dict(q=torch.zeros(2, 8, 128, dtype=BF), k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             lse=torch.zeros(2, 8), block_table=torch.zeros(2, 5, dtype=torch.int32),
             seqlens=torch.zeros(2, dtype=torch.int32), weights=torch.zeros(2, 4, 80), k_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.accumulate_kv_weights_paged(**a)


def _evict(**kw):
    a = dict(k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             block_table=torch.zeros(2, 3, dtype=torch.int32), seqlens=torch.zeros(2, dtype=torch.int32),
             weights=torch.zeros(2, 4, 48), new_block_table=torch.zeros(2, 2, dtype=torch.int32), budget=32, recent=4,
             k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.evict_kv_paged(**a)


def _cache(*shape, dtype=torch.int8):
    return torch.zeros(*shape, dtype=dtype)


CACHE_REFUSALS = [
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=torch.float16)), "bf16, float8_e4m3fn or int8"),
    (dict(k_cache=_cache(10, 16, 4)), r"\[num_pages, page_size, Hkv, D\]"),
    (dict(k_cache=_cache(10, 12, 4, 128)), "power of two"),
    (dict(k_cache=_cache(10, 16, 4, 64)), "head_dim must be 128"),
    (dict(k_cache=_cache(10, 16, 128, 4).transpose(2, 3)), "contiguous"),
    (dict(k_cache=_cache(10, 16, 4, 136)[..., :128]), "multiples of 16 bytes"),
    (dict(k_scale=torch.ones(10, 3)), "num_pages, Hkv"),
    (dict(k_scale=torch.ones(10, 4, dtype=torch.float64)), "fp32"),
    (dict(k_scale=1.0), "int8 caches need"),
]
BOTH_REFUSALS = CACHE_REFUSALS + [
    (dict(v_cache=_cache(10, 16, 4, 128, dtype=BF)), "share dtype and shape"),
    (dict(v_cache=_cache(9, 16, 4, 128)), "share dtype and shape"),
    (dict(v_scale=2.0), "int8 caches need"),
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8), v_scale=2.0),
     "both be tensors"),
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=BF), v_cache=_cache(10, 16, 4, 128, dtype=BF)), "no block scales"),
]
TABLE_REFUSALS = [
    (dict(block_table=torch.zeros(2, 5, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(3, 5, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 10, dtype=torch.int32)[:, ::2]), "block_table"),
    (dict(seqlens=torch.zeros(2, dtype=torch.int64)), "seqlens"),
]


@pytest.mark.parametrize("kw,text", BOTH_REFUSALS + TABLE_REFUSALS + [
    (dict(seqlens=torch.zeros(3, dtype=torch.int32)), "seqlens"),
    (dict(k=torch.zeros(2, 3, 4, 128)), "bf16 tokens"),
    (dict(v=torch.zeros(2, 2, 4, 128, dtype=BF)), "matching the caches"),
    (dict(k=torch.zeros(2, 3, 2, 128, dtype=BF), v=torch.zeros(2, 3, 2, 128, dtype=BF)), "matching the caches"),
    (dict(new_lens=torch.zeros(2, dtype=torch.int64)), "new_lens"),
    (dict(new_lens=torch.zeros(4, dtype=torch.int32)[::2]), "new_lens"),
    (dict(k_cache=_cache(1, 16, 4, 128).expand(10, 16, 4, 128)), "overlap itself"),
    (dict(v_scale=torch.ones(10, 1).expand(10, 4)), "overlap itself"),
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8), k_scale=0.0, v_scale=1.0),
     "positive"),
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8), k_scale=1.0,
          v_scale=float("nan")), "finite"),
    (dict(k_cache=_cache(10, 16, 4, 128, dtype=BF), v_cache=_cache(10, 16, 4, 128, dtype=BF), k_scale=2.0, v_scale=1.0),
     "no scale"),
    (dict(), "GPU"),
])
def test_append_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _append(**kw)


@pytest.mark.parametrize("kw,text", BOTH_REFUSALS + TABLE_REFUSALS + [
    (dict(q=torch.zeros(2, 8, 128)), "bf16 query"),
    (dict(q=torch.zeros(2, 1, 8, 128, dtype=BF)), "expected q"),
    (dict(q=torch.zeros(2, 6, 128, dtype=BF)), "divisible"),
    (dict(q=torch.zeros(2, 8, 64, dtype=BF)), "match Q"),
    (dict(seqlens=torch.zeros(3, dtype=torch.int32)), "seqlens"),
    (dict(max_seqlen=81), "max_seqlen"),
    (dict(max_seqlen=-1), "max_seqlen"),
    (dict(out=torch.zeros(2, 8, 128)), "out must be"),
    (dict(lse=torch.zeros(2, 8, dtype=torch.float64)), "lse must be"),
    (dict(), "GPU"),
])
def test_decode_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _decode(**kw)
    if kw != {}:
        with pytest.raises(ValueError, match=text):
            fg.prepare_decode_paged(**{**dict(
                q=torch.zeros(2, 8, 128, dtype=BF), k_cache=_cache(10, 16, 4, 128), v_cache=_cache(10, 16, 4, 128),
                block_table=torch.zeros(2, 5, dtype=torch.int32), seqlens=torch.zeros(2, dtype=torch.int32),
                k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4)), **kw})


@pytest.mark.parametrize("kw,text", CACHE_REFUSALS + TABLE_REFUSALS + [
    (dict(q=torch.zeros(2, 8, 128)), "bf16 query"),
    (dict(q=torch.zeros(2, 6, 128, dtype=BF)), "divisible"),
    (dict(lse=torch.zeros(2, 7)), "lse must be"),
    (dict(lse=torch.zeros(8, 2).t()), "lse must be"),
    (dict(weights=torch.zeros(2, 4, 80, dtype=torch.float64)), "weights must be"),
    (dict(weights=torch.zeros(2, 3, 80)), "weights must be"),
    (dict(weights=torch.zeros(2, 4, 160)[:, :, ::2]), "weights must be"),
    (dict(weights=torch.zeros(1, 4, 80).expand(2, 4, 80)), "overlap itself"),
    (dict(weights=torch.zeros(2, 4, 70), max_seqlen=75), "hold max_seqlen"),
    (dict(max_seqlen=81, weights=torch.zeros(2, 4, 99)), "max_seqlen"),
    (dict(), "GPU"),
])
def test_weights_refuse(kw, text):
    with pytest.raises(ValueError, match=text):
        _weights(**kw)


@pytest.mark.parametrize("kw,text", BOTH_REFUSALS + [
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(seqlens=torch.zeros(2, dtype=torch.int64)), "seqlens"),
    (dict(seqlens=torch.zeros(2, 1, dtype=torch.int32)), "seqlens"),
    (dict(new_block_table=torch.zeros(2, 1, dtype=torch.int32)), "pages for"),
    (dict(new_block_table=torch.zeros(1, 2, dtype=torch.int32)), "new_block_table"),
    (dict(budget=0), "budget"),
    (dict(recent=-1), "recent"),
    (dict(weights=torch.zeros(2, 5, 48)), "weights must be"),
    (dict(weights=torch.zeros(2, 4, 40), max_seqlen=41), "hold max_seqlen"),
    (dict(max_seqlen=49, weights=torch.zeros(2, 4, 60)), "max_seqlen"),
    (dict(new_weights=torch.zeros(2, 4, 47)), "weights' shape"),
    (dict(new_weights=torch.zeros(1, 4, 48).expand(2, 4, 48)), "overlap itself"),
    (dict(kept=torch.zeros(2, 4, 32, dtype=torch.int64)), "kept must be"),
    (dict(kept=torch.zeros(2, 4, 31, dtype=torch.int32)), "kept must be"),
    (dict(new_seqlens=torch.zeros(3, dtype=torch.int32)), "new_seqlens"),
    (dict(k_cache=_cache(1, 16, 4, 128).expand(10, 16, 4, 128)), "overlap itself"),
    (dict(), "GPU"),
])
def test_evict_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _evict(**kw)


def test_evict_refuses_outputs_over_inputs():
    w = torch.zeros(2, 4, 48)
    with pytest.raises(ValueError, match="apart"):
        _evict(weights=w, new_weights=w)
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="apart"):
        _evict(seqlens=lens, new_seqlens=lens)
    wide = torch.zeros(2 * 4 * 48 + 10, dtype=torch.float32)
    with pytest.raises(ValueError, match="apart"):
        _evict(weights=wide[:384].view(2, 4, 48), new_weights=wide[10:].view(2, 4, 48))


def test_refuses_written_tensors_over_others():
    k = _cache(10, 16, 4, 128)
    with pytest.raises(ValueError, match="apart"):
        _append(k_cache=k, v_cache=k)
    with pytest.raises(ValueError, match="apart"):
        _evict(k_cache=k, v_cache=k)
    k = _cache(10, 16, 4, 128, dtype=BF)
    with pytest.raises(ValueError, match="apart"):
        _append(k=k[:2, :3], k_cache=k, v_cache=k.clone(), k_scale=1.0, v_scale=1.0)
    both = _cache(10, 2, 16, 4, 128)   # interleaved caches are two memories
    with pytest.raises(ValueError, match="GPU"):
        _append(k_cache=both[:, 0], v_cache=both[:, 1])
    w = torch.zeros(2, 4, 80)
    with pytest.raises(ValueError, match="apart"):
        _weights(weights=w, lse=w[0, 0, :16].view(2, 8))
    with pytest.raises(ValueError, match="overlap itself"):
        _decode(out=torch.zeros(1, 8, 128, dtype=BF).expand(2, 8, 128))


def test_scales_that_stand_for_a_number():
    """Tensors of one element beside an fp8 cache of more blocks stay numbers; a cache
    of one block takes them as its scales."""
    c = _cache(10, 16, 4, 128, dtype=F8)
    one = torch.tensor(0.5)
    for s in (one, one.view(1), one.view(1, 1)):
        assert not flash_gqa._has_block_scales(c, s, s)
        assert not flash_gqa._has_block_scales(c, 1.0, s)
    assert flash_gqa._has_block_scales(c[:1, :, :1], one.view(1, 1), one.view(1, 1))
    assert flash_gqa._has_block_scales(c, torch.ones(10, 4), torch.ones(10, 4))
    assert flash_gqa._has_block_scales(_cache(10, 16, 4, 128), 1.0, 1.0)
    assert not flash_gqa._has_block_scales(c, 0.5, 2)


def test_c_abi_refuses_null_arguments():
    L = _lib.lib()
    for name in ("fgqa_kv_append", "fgqa_decode_blocks", "fgqa_kv_weights", "fgqa_kv_evict"):
        f = getattr(L, name)
        f.restype = ctypes.c_int
        f.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
        assert f(None, None) == _lib.FGQA_ERR_INVALID_ARGUMENT


def test_arguments_of_other_types():
    """What is no tensor, number or whole number; too large numbers; sparse tensors; wrong argument counts."""
    with pytest.raises(TypeError, match="block_table must be a tensor"):
        _append(block_table=[[0]])
    with pytest.raises(TypeError):
        _append(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8), k_scale="1", v_scale=1.0)
    with pytest.raises(TypeError):
        _weights(max_seqlen=[3])
    with pytest.raises(ValueError, match="budget"):
        _evict(budget=2 ** 40)
    with pytest.raises(ValueError, match="budget"):
        _evict(budget=2 ** 80)
    with pytest.raises(ValueError, match="finite"):
        _append(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8), k_scale=1e300, v_scale=1.0)
    with pytest.raises(ValueError, match="split_tokens"):
        _decode(split_tokens=-1)
    with pytest.raises((RuntimeError, ValueError)):
        _append(block_table=torch.zeros(2, 5, dtype=torch.int32).to_sparse())
    with pytest.raises(TypeError, match="arguments"):
        fg.native().append(1, 2)


def test_calls_for_another_device(monkeypatch):
    """A call whose tensors live on another device runs again with that one current."""
    seen, now = [], [0]

    class Native:
        @staticmethod
        def append(*args):
            seen.append((now[0], args))
            return NotImplemented if now[0] != 1 else None

    class Current:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            now[0] = self.device

        def __exit__(self, *_):
            now[0] = 0

    class On1:
        device = 1

    monkeypatch.setattr(_lib, "native", lambda: Native)
    monkeypatch.setattr(torch.cuda, "device", Current)
    assert kv_cache.call_native("append", On1, 3, 4) is None
    assert seen == [(0, (3, 4)), (1, (3, 4))] and now == [0]
