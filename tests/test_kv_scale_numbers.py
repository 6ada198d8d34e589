"""CPU tests: a tensor of one element as k_scale or v_scale means the same to every
function of the paged cache: a number, or all block scales of a cache of one page and
head."""
import pytest
import torch

from cuda_llm_ops_amd import flash_gqa
from tests.test_kv_host import BF, F8, _append, _cache, _decode, _evict, _weights

F8S = dict(k_cache=_cache(10, 16, 4, 128, dtype=F8), v_cache=_cache(10, 16, 4, 128, dtype=F8))
ONE = torch.tensor(0.5)


@pytest.mark.parametrize("call", [_append, _evict, _decode])
@pytest.mark.parametrize("s", [ONE, ONE.view(1), ONE.view(1, 1), ONE.double()])
def test_one_element_is_a_number(call, s):
    for v in (s, 0.25, s.clone()):
        with pytest.raises(ValueError, match="GPU"):
            call(**F8S, k_scale=s, v_scale=v)
        with pytest.raises(ValueError, match="GPU"):
            call(**F8S, k_scale=v, v_scale=s)
    with pytest.raises(ValueError, match="GPU"):
        _weights(k_cache=F8S["k_cache"], k_scale=s)


def test_numbers_are_checked():
    with pytest.raises(ValueError, match="positive"):
        _append(**F8S, k_scale=-ONE, v_scale=ONE)
    with pytest.raises(ValueError, match="finite"):
        _append(**F8S, k_scale=ONE / 0, v_scale=ONE)
    with pytest.raises(ValueError, match="num_pages, Hkv"):
        _append(**F8S, k_scale=ONE, v_scale=torch.ones(10, 4))
    with pytest.raises(ValueError, match="int8 caches need|num_pages, Hkv"):
        _append(k_scale=ONE, v_scale=ONE)
    bf = dict(k_cache=_cache(10, 16, 4, 128, dtype=BF), v_cache=_cache(10, 16, 4, 128, dtype=BF))
    with pytest.raises(ValueError, match="no scale"):
        _append(**bf, k_scale=ONE, v_scale=ONE)
    with pytest.raises(ValueError, match="GPU"):
        _append(**bf, k_scale=2 * ONE, v_scale=1.0)


def test_a_cache_of_one_block():
    one = torch.ones(1, 1)
    f8, bf, i8 = (_cache(1, 16, 1, 128, dtype=t) for t in (F8, BF, torch.int8))
    has = flash_gqa._has_block_scales
    assert has(f8, one, one) and has(i8, one, one)
    # what is not all block scales stays a number, as with larger caches
    assert not has(f8, one, 1.0) and not has(f8, 1.0, one) and not has(f8, one.double(), one.double())
    assert not has(f8, one.view(1), one.view(1)) and not has(f8, one, one.to("meta"))
    assert not has(bf, one, one)
    kw = dict(k=torch.zeros(2, 3, 1, 128, dtype=BF), v=torch.zeros(2, 3, 1, 128, dtype=BF), v_cache=f8.clone(), k_cache=f8)
    with pytest.raises(ValueError, match="k_scale and v_scale must be apart"):   # block scales
        _append(**kw, k_scale=one, v_scale=one)
    for k, v in ((one, 1.0), (1.0, one), (one.double(), one.double()), (one.view(1), one)):
        with pytest.raises(ValueError, match="GPU"):
            _append(**kw, k_scale=k, v_scale=v)
