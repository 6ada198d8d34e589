"""CPU tests of the decode of sequences that begin alike: every refusal of the Python
function, and the bounds of its cuts under sanitizers."""
import os
import shutil

import pytest
import torch

import cuda_llm_ops_amd as fg
from tests.test_host_sanitizers import HOST, ROOT, _build_and_run

BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_shared_plan_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_shared_plan", [os.path.join(HOST, n) for n in (
        "fgqa_plan.cpp", "kv_plan.cpp", "pages_plan.cpp")] + [os.path.join(ROOT, "tests", "host", "test_shared_plan.cpp")])


def _decode(**kw):
    a = dict(q=torch.zeros(2, 8, 128, dtype=BF), k_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8),
             v_cache=torch.zeros(10, 16, 4, 128, dtype=torch.int8), block_table=torch.zeros(2, 5, dtype=I32),
             seqlens=torch.zeros(2, dtype=I32), group_starts=torch.tensor([0, 2], dtype=I32),
             shared_lens=torch.tensor([16], dtype=I32), k_scale=torch.ones(10, 4), v_scale=torch.ones(10, 4))
    a.update(kw)
    return fg.decode_flash_gqa_paged_shared(**a)


@pytest.mark.parametrize("kw,text", [
    (dict(q=torch.zeros(2, 8, 128)), "bf16 query"),
    (dict(q=torch.zeros(2, 1, 8, 128, dtype=BF)), "expected q"),
    (dict(q=torch.zeros(2, 6, 128, dtype=BF)), "divisible"),
    (dict(q=torch.zeros(2, 8, 64, dtype=BF)), "match Q"),
    (dict(k_cache=torch.zeros(10, 16, 4, 64, dtype=torch.int8), v_cache=torch.zeros(10, 16, 4, 64, dtype=torch.int8)),
     "head_dim must be 128"),
    (dict(k_scale=1.0), "int8 caches need"),
    (dict(block_table=torch.zeros(3, 5, dtype=I32)), "block_table"),
    (dict(seqlens=torch.zeros(2, dtype=torch.int64)), "seqlens"),
    (dict(shared_lens=torch.zeros(1, dtype=torch.int64)), "shared_lens"),
    (dict(shared_lens=torch.zeros(1, 1, dtype=I32)), "shared_lens"),
    (dict(group_starts=torch.zeros(1, dtype=I32)), "group_starts"),
    (dict(group_starts=torch.zeros(4, dtype=I32)[::2]), "group_starts"),
    (dict(group_starts=torch.zeros(4098, dtype=I32), shared_lens=torch.zeros(4097, dtype=I32)), "4096 groups"),
    (dict(max_seqlen=81), "max_seqlen"),
    (dict(max_seqlen=-1), "max_seqlen"),
    (dict(out=torch.zeros(2, 8, 128)), "out must be"),
    (dict(out=torch.zeros(1, 8, 128, dtype=BF).expand(2, 8, 128)), "overlap itself"),
    (dict(lse=torch.zeros(2, 8, dtype=torch.float64)), "lse must be"),
    (dict(workspace=torch.zeros(8, 8).t()), "workspace must be contiguous"),
    (dict(), "GPU"),
])
def test_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _decode(**kw)


def test_refuses_outputs_over_inputs():
    q = torch.zeros(2, 8, 128, dtype=BF)
    with pytest.raises(ValueError, match="apart"):
        _decode(q=q, out=q)
    k = torch.zeros(10, 16, 4, 128, dtype=torch.int8)
    with pytest.raises(ValueError, match="apart"):
        _decode(k_cache=k, out=k.view(-1)[:4096].view(BF).view(2, 8, 128))
    s = torch.ones(10, 4)
    with pytest.raises(ValueError, match="apart"):
        _decode(k_scale=s, lse=s.view(-1)[:16].view(2, 8))
    with pytest.raises(ValueError, match="apart"):
        _decode(out=q, workspace=q)
    with pytest.raises(TypeError, match="shared_lens must be a tensor"):
        _decode(shared_lens=[16])
