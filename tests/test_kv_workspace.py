"""CPU tests: a workspace whose elements are not all there (an expanded one) or that is
no GPU memory is refused."""
import pytest
import torch

import cuda_llm_ops_amd as fg
from cuda_llm_ops_amd import flash_gqa
from tests.test_kv_host import BF, _cache, _decode


@pytest.mark.parametrize("work", [torch.empty(1, dtype=torch.uint8).expand(1 << 30),
                                  torch.empty(1 << 12, 2, dtype=torch.uint8)[:, 0]])
def test_not_contiguous(work):
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        _decode(workspace=work)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        fg.prepare_decode_paged(torch.zeros(2, 8, 128, dtype=BF), _cache(10, 16, 4, 128), _cache(10, 16, 4, 128),
                                torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                                k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4), workspace=work)
    with pytest.raises(ValueError, match="GPU"):
        flash_gqa._workspace(work)


def test_other_paths(monkeypatch):
    assert flash_gqa._workspace(None) == (0, 0)
    with pytest.raises(ValueError, match="GPU"):
        flash_gqa._workspace(torch.empty(100))
    monkeypatch.setattr(flash_gqa, "_require_cuda", lambda *ts: None)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        flash_gqa._workspace(torch.empty(1).expand(1 << 30))
    w = torch.empty(100)
    assert flash_gqa._workspace(w) == (w.data_ptr(), 400)


def test_contiguous_ones_get_as_far_as_the_device():
    with pytest.raises(ValueError, match="GPU"):
        _decode(workspace=torch.empty(1 << 12, dtype=torch.uint8))
