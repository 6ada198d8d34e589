"""CPU tests: outputs of the paged cache's operators over what the same call reads or
writes are refused."""
import os
import shutil

import pytest
import torch

from tests.test_host_sanitizers import HOST, ROOT, _build_and_run
from tests.test_kv_host import _cache, _evict, _weights


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_c_abi_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_kv_in_place",
                   [os.path.join(HOST, "fgqa_plan.cpp"), os.path.join(HOST, "kv_plan.cpp"),
                    os.path.join(ROOT, "tests", "host", "test_kv_in_place.cpp")])


@pytest.mark.parametrize("what", ["k_cache", "v_cache", "k_scale", "v_scale"])
def test_evict_outputs_over_the_cache(what):
    k, v = _cache(10, 16, 4, 128), _cache(10, 16, 4, 128)
    s = [torch.ones(200, 4) for _ in range(2)]
    kw = dict(k_cache=k, v_cache=v, k_scale=s[0][:10], v_scale=s[1][:10])
    under = {"k_cache": k.view(torch.float32).view(-1), "v_cache": v.view(torch.float32).view(-1),
             "k_scale": s[0].view(-1)[4:], "v_scale": s[1].view(-1)[36:]}[what]
    with pytest.raises(ValueError, match="apart"):
        _evict(**kw, new_weights=under[:384].view(2, 4, 48))
    with pytest.raises(ValueError, match="apart"):
        _evict(**kw, weights=under[:384].view(2, 4, 48))
    with pytest.raises(ValueError, match="apart"):
        _evict(**kw, kept=under[:256].view(2, 4, 32).view(torch.int32))
    with pytest.raises(ValueError, match="apart"):
        _evict(**kw, new_seqlens=under[:2].view(torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        _evict(**kw)


def test_weights_over_the_cache():
    k, s = _cache(10, 16, 4, 128), torch.ones(200, 4)
    for under in (k.view(torch.float32).view(-1), s.view(-1)):
        with pytest.raises(ValueError, match="apart"):
            _weights(k_cache=k, k_scale=s[:10], weights=under[:640].view(2, 4, 80))
