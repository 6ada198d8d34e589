"""CPU tests of the norm and rotation's host side: refusals of the Python functions
(before any GPU is looked at), the C ABI's exports and statuses, the test of blocks that
share memory, and the reference's gradients against differences."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

import cuda_llm_ops_amd as fg
from cuda_llm_ops_amd import _lib
from tests import _rope_reference as ref
from tests.test_host_sanitizers import HOST, ROOT, _build_and_run

BF = torch.bfloat16


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rope_plan_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_rope_plan", [os.path.join(HOST, "rope_plan.cpp"),
                                                os.path.join(ROOT, "tests", "host", "test_rope_plan.cpp")])


def test_exported():
    names = set(re.findall(r"^int (fgqa_\w+)\(", open(os.path.join(ROOT, "include", "fgqa_rope.h")).read(), flags=re.M))
    assert names == {"fgqa_qk_norm_rope", "fgqa_qk_norm_rope_backward", "fgqa_qk_norm_rope_backward_workspace_bytes"}
    syms = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], check=True, capture_output=True, text=True).stdout
    for n in names:
        assert re.search(rf"\bT {n}$", syms, flags=re.M), n


def test_c_abi_refuses_null_arguments():
    L = ctypes.CDLL(_lib.LIB_PATH)
    for name in ("fgqa_qk_norm_rope", "fgqa_qk_norm_rope_backward"):
        f = getattr(L, name)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
        assert f(None, None) == _lib.FGQA_ERR_INVALID_ARGUMENT


def _forward(**kw):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF), k=torch.zeros(2, 3, 2, 64, dtype=BF),
             positions=torch.zeros(2, 3, dtype=torch.int32), inv_freq=torch.ones(32), q_weight=torch.ones(64, dtype=BF),
             k_weight=torch.ones(64, dtype=BF))
    a.update(kw)
    return fg.qk_norm_rope(**a)


def _backward(**kw):
    a = dict(grad_q=torch.zeros(2, 3, 4, 64, dtype=BF), grad_k=torch.zeros(2, 3, 2, 64, dtype=BF),
             q=torch.zeros(2, 3, 4, 64, dtype=BF), k=torch.zeros(2, 3, 2, 64, dtype=BF),
             positions=torch.zeros(2, 3, dtype=torch.int32), inv_freq=torch.ones(32), q_weight=torch.ones(64, dtype=BF),
             k_weight=torch.ones(64, dtype=BF))
    a.update(kw)
    return fg.qk_norm_rope_backward(**a)


BOTH = [
    (dict(positions=torch.zeros(2, 3)), "int32 or int64"),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int32)), "match the tokens"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int32)), "match the tokens"),
    (dict(positions=torch.zeros((), dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros(1, 1, 2, 3, dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros(0, 2, 3, dtype=torch.int32), axes=torch.zeros(32, dtype=torch.int32)), "at least one axis"),
    (dict(positions=torch.zeros(3, 2, 3, dtype=torch.int32)), "need axes"),
    (dict(axes=torch.zeros(31, dtype=torch.int32)), "axes must be"),
    (dict(axes=torch.zeros(32, dtype=torch.int64)), "axes must be"),
    (dict(inv_freq=torch.ones(33)), "multiple of 8"),
    (dict(inv_freq=torch.ones(40)), "at most half"),
    (dict(inv_freq=torch.ones(32, dtype=torch.float64)), "fp32"),
    (dict(inv_freq=torch.ones(64)[::2]), "contiguous fp32"),
    (dict(inv_freq=None), "both be given"),
    (dict(positions=None, inv_freq=None, axes=torch.zeros(32, dtype=torch.int32)), "need positions"),
    (dict(k_weight=None), "both be given"),
    (dict(k_weight=torch.ones(64)), "both bf16 or both fp32"),
    (dict(q_weight=torch.ones(32, dtype=BF)), r"\[D\]"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(), "GPU"),
]


@pytest.mark.parametrize("kw,text", BOTH + [
    (dict(q=torch.zeros(2, 3, 4, 64)), "must be bf16"),
    (dict(k=torch.zeros(2, 4, 2, 64, dtype=BF)), "all but their heads"),
    (dict(k=torch.zeros(2, 3, 64, dtype=BF)), "both be"),
    (dict(k=torch.zeros(2, 3, 0, 64, dtype=BF)), "must have heads"),
    (dict(q=torch.zeros(2, 3, 4, 72, dtype=BF), k=torch.zeros(2, 3, 2, 72, dtype=BF)), "multiple of 16"),
    (dict(q=torch.zeros(2, 3, 4, 272, dtype=BF), k=torch.zeros(2, 3, 2, 272, dtype=BF)), "up to 256"),
    (dict(q_out=torch.zeros(2, 3, 4, 64)), "q_out must be bf16"),
    (dict(k_out=torch.zeros(2, 3, 4, 64, dtype=BF)), "k_out must be bf16"),
    (dict(q_out=torch.zeros(1, 3, 4, 64, dtype=BF).expand(2, 3, 4, 64)), "overlap itself"),
    (dict(q_out=torch.zeros(2, 3, 4, 68, dtype=BF)[..., :64]), "16-byte aligned"),
])
def test_forward_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _forward(**kw)


@pytest.mark.parametrize("kw,text", BOTH + [
    (dict(grad_q=torch.zeros(2, 3, 4, 64)), "must be bf16"),
    (dict(q=torch.zeros(2, 3, 5, 64, dtype=BF)), "q's and k's shapes"),
    (dict(k=torch.zeros(2, 3, 2, 48, dtype=BF)), "all but their heads"),
])
def test_backward_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _backward(**kw)


def test_refuses_other_types():
    with pytest.raises(TypeError, match="q must be a tensor"):
        _forward(q=[1])
    with pytest.raises(TypeError, match="k must be a tensor"):
        _backward(k=None)
    with pytest.raises(TypeError):
        _forward(eps="1")


def test_outputs_over_inputs():
    """In place is a call like any other; every other overlap is refused."""
    qkv = torch.zeros(2, 3, 8, 64, dtype=BF)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    for kw in (dict(q_out=q, k_out=k), dict(q_out=q), dict(k_out=k), dict(k_out=v)):
        with pytest.raises(ValueError, match="GPU"):
            _forward(q=q, k=k, **kw)
    for kw in (dict(q_out=qkv[:, :, 1:5]), dict(k_out=qkv[:, :, 3:5]), dict(k_out=q[:, :, :2]), dict(k_out=qkv[:, :, 5:7]),
               dict(q_out=qkv[:, :, 4:]), dict(q_out=qkv.view(-1)[8:8 + 1536].view(2, 3, 4, 64))):
        with pytest.raises(ValueError, match="apart"):
            _forward(q=q, k=k, **kw)
    w = torch.zeros(2 * 3 * 4 * 64, dtype=BF)
    with pytest.raises(ValueError, match="apart from positions"):
        _forward(q_out=w.view(2, 3, 4, 64), q_weight=w[:64])


def test_reference_gradients_against_differences():
    """The formula's gradients of a random sum of outputs against central differences in float64."""
    g = np.random.default_rng(1)
    x, w, dy = g.normal(size=(3, 2, 16)), g.normal(size=16), g.normal(size=(3, 2, 16))
    theta = ref.angles(np.array([[3, 70, 5], [1, 2, 900]]), 1.0 / 3 ** np.arange(6), np.array([0, 1, 1, 0, 1, 0]))

    def loss(x, w, inter):
        return (ref.forward(x, w, theta, 1e-3, inter)[0] * dy).sum()

    for inter in (False, True):
        dx, _, dw, _ = ref.backward(dy, x, w, theta, 1e-3, inter)
        h = 1e-6   # (differences are off by about h^2 and 2^-53 / h)
        for i in np.ndindex(x.shape):
            e = np.zeros_like(x)
            e[i] = h
            assert abs((loss(x + e, w, inter) - loss(x - e, w, inter)) / (2 * h) - dx[i]) < 1e-7
        for i in range(16):
            e = np.zeros_like(w)
            e[i] = h
            assert abs((loss(x, w + e, inter) - loss(x, w - e, inter)) / (2 * h) - dw[i]) < 1e-7
