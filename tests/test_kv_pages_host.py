"""CPU tests of forking and compacting: exports and statuses of the C ABI, the host
validation under sanitizers, every refusal of the Python functions, the reference's own rules."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import cuda_llm_ops_amd as fg
from cuda_llm_ops_amd import _lib
from tests import _pages_reference as ref
from tests.test_host_sanitizers import HOST, ROOT, _build_and_run

BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_pages_plan_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_pages_plan", [os.path.join(HOST, n) for n in (
        "fgqa_plan.cpp", "kv_plan.cpp", "pages_plan.cpp")] + [os.path.join(ROOT, "tests", "host", "test_pages_plan.cpp")])


def test_exported():
    names = set(re.findall(r"^int (fgqa_\w+)\(", open(os.path.join(ROOT, "include", "fgqa_pages.h")).read(), flags=re.M))
    assert {"fgqa_kv_fork", "fgqa_kv_fork_workspace_bytes", "fgqa_kv_compact", "fgqa_kv_compact_workspace_bytes"} <= names
    syms = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], check=True, capture_output=True, text=True).stdout
    L = ctypes.CDLL(_lib.LIB_PATH)
    for n in names:
        assert re.search(rf"\bT {n}$", syms, flags=re.M), n
        f = getattr(L, n)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
        assert f(None, None) == _lib.FGQA_ERR_INVALID_ARGUMENT


def _fork(**kw):
    a = dict(k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             block_table=torch.zeros(2, 5, dtype=I32), seqlens=torch.zeros(2, dtype=I32), k_scale=torch.ones(10, 4),
             v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.fork_kv_paged(**a)


def _compact(**kw):
    a = dict(k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             block_table=torch.zeros(2, 5, dtype=I32), seqlens=torch.zeros(2, dtype=I32), k_scale=torch.ones(10, 4),
             v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.compact_kv_paged(**a)


def _c(*shape, dtype=torch.int8):
    return torch.zeros(*shape, dtype=dtype)


BOTH = [
    (dict(k_cache=_c(10, 16, 4, 128, dtype=torch.float16)), "bf16, float8_e4m3fn or int8"),
    (dict(v_cache=_c(9, 16, 4, 128)), "share dtype and shape"),
    (dict(k_scale=torch.ones(10, 3)), "num_pages, Hkv"),
    (dict(k_scale=1.0), "int8 caches need"),
    (dict(k_cache=_c(1, 16, 4, 128).expand(10, 16, 4, 128)), "overlap itself"),
    (dict(v_scale=torch.ones(10, 1).expand(10, 4)), "overlap itself"),
    (dict(block_table=torch.zeros(2, 5, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(3, 5, dtype=I32)), "block_table"),
    (dict(seqlens=torch.zeros(2, 1, dtype=I32)), "seqlens"),
    (dict(seqlens=torch.zeros(2, dtype=torch.int64)), "seqlens"),
    (dict(held=torch.zeros(9, dtype=torch.bool)), "held must be"),
    (dict(held=torch.zeros(10, dtype=I32)), "held must be"),
    (dict(new_block_table=torch.zeros(2, 5, dtype=torch.int64)), "new_block_table"),
    (dict(new_block_table=torch.zeros(1, 5, dtype=I32).expand(2, 5)), "overlap itself"),
    (dict(), "GPU"),
]


@pytest.mark.parametrize("kw,text", BOTH + [
    (dict(parents=torch.zeros(3, dtype=torch.int64)), "parents must be"),
    (dict(parents=torch.zeros(3, 1, dtype=I32)), "parents must be"),
    (dict(parents=torch.zeros(6, dtype=I32)[::2]), "parents must be"),
    (dict(new_lens=torch.zeros(3, dtype=I32)), "new_lens must be"),
    (dict(parents=torch.zeros(3, dtype=I32), new_lens=torch.zeros(2, dtype=I32)), "new_lens must be"),
    (dict(max_pages=-1), "max_pages"),
    (dict(max_pages=4, new_block_table=torch.zeros(2, 5, dtype=I32)), "max_pages columns"),
    (dict(parents=torch.zeros(3, dtype=I32), new_block_table=torch.zeros(2, 5, dtype=I32)), "new_block_table"),
    (dict(new_seqlens=torch.zeros(3, dtype=I32)), "new_seqlens"),
    (dict(num_free=torch.zeros(2, dtype=I32)), "num_free"),
])
def test_fork_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _fork(**kw)


@pytest.mark.parametrize("kw,text", BOTH + [
    (dict(new_block_table=torch.zeros(2, 4, dtype=I32)), "block_table's shape"),
    (dict(num_used=torch.zeros(1)), "num_used"),
])
def test_compact_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _compact(**kw)


def test_outputs_over_inputs():
    t, n = torch.zeros(2, 5, dtype=I32), torch.zeros(2, dtype=I32)
    for f in (_fork, _compact):
        with pytest.raises(ValueError, match="apart"):
            f(block_table=t, new_block_table=t)
        k = _c(10, 16, 4, 128)
        with pytest.raises(ValueError, match="apart"):
            f(k_cache=k, v_cache=k)
        with pytest.raises(ValueError, match="apart"):
            f(k_cache=k, block_table=k.view(I32).view(-1)[:10].view(2, 5))
    with pytest.raises(ValueError, match="apart"):
        _fork(seqlens=n, new_seqlens=n)
    with pytest.raises(ValueError, match="apart"):
        _fork(new_lens=n, new_seqlens=n)
    with pytest.raises(ValueError, match="apart"):
        _fork(new_block_table=t, num_free=t[0, :1])
    with pytest.raises(ValueError, match="apart"):
        _compact(new_block_table=t, num_used=t[1, 3:4])
    with pytest.raises(TypeError, match="seqlens must be a tensor"):
        _fork(seqlens=[1, 2])


def test_reference_rules():
    """Worked by hand: two children of a partly filled row, a dropped row whose pages are free at once."""
    table, lens = [[4, 7, -1], [2, -1, -1], [0, 1, 9]], [20, 16, 40]
    new, n, copies, left = ref.fork(table, lens, 16, 10, [0, 0, 1, -1], [1, 13, 1, 0])
    # rows 0 and 1 share page 4; 7 stays with row 0; row 2's old pages (0, 1, 9) are free
    assert new == [[4, 7, -1], [4, 0, 1], [2, 3, -1], [-1, -1, -1]]
    assert n == [20, 20, 16, 0] and copies == [(7, 0, 4)] and left == 4
    # in use: 0, 2, 4 and 7 (pages 1 and 3 are for tokens to come); 4 and 7 move to 1 and 3
    new, moves, used = ref.compact(new, n, 16, 10)
    assert new == [[1, 3, -1], [1, 0, -1], [2, -1, -1], [-1, -1, -1]]
    assert moves == [(4, 1), (7, 3)] and used == 4
