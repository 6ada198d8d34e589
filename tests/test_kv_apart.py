"""CPU tests: calls that write a paged cache refuse K and V caches, or block scales,
that share memory, and take interleaved ones."""
import os
import shutil

import pytest
import torch

from tests.test_host_sanitizers import HOST, ROOT, _build_and_run
from tests.test_kv_host import _append, _cache, _decode, _evict


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_views_and_c_abi_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_kv_apart",
                   [os.path.join(HOST, "fgqa_plan.cpp"), os.path.join(HOST, "kv_plan.cpp"),
                    os.path.join(ROOT, "tests", "host", "test_kv_apart.cpp")])


@pytest.mark.parametrize("call", [_append, _evict])
def test_shared_scales(call):
    s = torch.ones(10, 4)
    with pytest.raises(ValueError, match="k_scale and v_scale must be apart"):
        call(k_scale=s, v_scale=s)
    s = torch.ones(15, 4)
    with pytest.raises(ValueError, match="k_scale and v_scale must be apart"):
        call(k_scale=s[:10], v_scale=s[5:])
    s = torch.ones(11, 4, 2)
    with pytest.raises(ValueError, match="k_scale and v_scale must be apart"):
        call(k_scale=s[:10, :, 0], v_scale=s.view(-1)[2:].as_strided((10, 4), (8, 2)))
    s = s[:10]
    with pytest.raises(ValueError, match="GPU"):      # interleaved: apart
        call(k_scale=s[:, :, 0], v_scale=s[:, :, 1])
    s = torch.ones(10, 2, 4)
    with pytest.raises(ValueError, match="GPU"):
        call(k_scale=s[:, 0], v_scale=s[:, 1])


@pytest.mark.parametrize("call", [_append, _evict])
def test_shared_caches(call):
    k = _cache(15, 16, 4, 128)
    with pytest.raises(ValueError, match="k_cache and v_cache must be apart"):
        call(k_cache=k[:10], v_cache=k[5:])
    k = _cache(10, 16, 6, 128)
    with pytest.raises(ValueError, match="k_cache and v_cache must be apart"):
        call(k_cache=k[:, :, :4], v_cache=k[:, :, 2:])
    for both in (_cache(10, 16, 8, 128), _cache(10, 32, 4, 128)):
        k, v = (both[:, :, :4], both[:, :, 4:]) if both.shape[1] == 16 else (both[:, :16], both[:, 16:])
        with pytest.raises(ValueError, match="GPU"):
            call(k_cache=k, v_cache=v)


def test_a_decode_takes_one_scale_tensor_for_both():
    s = torch.ones(10, 4)
    with pytest.raises(ValueError, match="GPU"):
        _decode(k_scale=s, v_scale=s)
