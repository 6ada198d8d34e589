"""Norm and rotation, and their gradients, over more bytes of rows than the caches hold, which are read and written
past them (2^28 bytes in all: 2^26 elements of the forward, or the gradients without weights, and 2^28 / 6 of those
with): bit for bit as over slices of the tokens that stay below, rows of them and the weights'
gradients against float64."""
import numpy as np
import pytest

from tests import _rope_reference as ref
from tests.test_gpu_qk_rope import _check_backward, _check_forward, _make

pytestmark = pytest.mark.gpu

CASES = [
    # lead, Hq, Hkv, D, R, axes, interleaved, weights: a little more than 2^26 elements each
    ((1, 16391), 24, 8, 128, 128, None, False, "bf16"),
    ((3, 5471), 24, 8, 128, 96, 3, True, "fp32"),
    ((1, 26220), 8, 2, 256, 256, None, False, None),
    ((32775,), 28, 4, 64, 64, 2, True, None),
    ((1, 41950), 17, 3, 80, 48, None, False, "bf16"),
    ((1, 16391), 24, 8, 128, 64, None, False, None),
]
IDS = [f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[6]}-{c[7]}" for c in CASES]


def _tokens(c, at):
    """The call of some tokens: `at` indexes the token dim, the last of the leading ones."""
    out = dict(c)
    out["q"], out["k"] = c["q"][..., at, :, :], c["k"][..., at, :, :]
    out["positions"] = c["positions"][..., at]
    return out


def _slices(n):
    """Two parts, each below the caches' bytes and of more than a wave for each SIMD."""
    return [slice(0, n // 2 + 3), slice(n // 2 + 3, n)]


def _same(torch, whole, parts, at):
    return all(torch.equal(whole[..., s, :, :], p) for s, p in zip(at, parts))


@pytest.mark.parametrize("lead,Hq,Hkv,D,R,axes,interleaved,weights", CASES, ids=IDS)
def test_forward(cuda, lead, Hq, Hkv, D, R, axes, interleaved, weights):
    import torch
    import cuda_llm_ops_amd as fg
    print(lead, Hq, Hkv, D, R, axes, interleaved, weights, flush=True)
    n = lead[-1]
    assert int(np.prod(lead)) * (Hq + Hkv) * D > 1 << 26
    c = _make(torch, cuda, lead, Hq, Hkv, D, R, axes=axes, weights=weights)
    outs = fg.qk_norm_rope(**c, interleaved=interleaved)
    at = _slices(n)
    parts = [fg.qk_norm_rope(**_tokens(c, s), interleaved=interleaved) for s in at]
    for i in range(2):
        assert _same(torch, outs[i], [p[i] for p in parts], at)
    some = torch.tensor([0, 1, n // 2 + 2, n // 2 + 3, n - 2, n - 1] + list(range(5, n, n // 50)), device=cuda)
    _check_forward(_tokens(c, some), [o[..., some, :, :] for o in outs], interleaved=interleaved)
    # in place: v's rows, between the heads that are written, stay as they are
    rest = c["q"]._base[..., Hq + Hkv:, :].clone()
    fg.qk_norm_rope(**c, interleaved=interleaved, q_out=c["q"], k_out=c["k"])
    assert torch.equal(c["q"], outs[0]) and torch.equal(c["k"], outs[1])
    assert torch.equal(c["q"]._base[..., Hq + Hkv:, :], rest)


def _weight_sums(torch, c, grads, interleaved):
    """(of q_weight, its bound, of k_weight, its bound) over all rows, some tokens at a time."""
    out = []
    n = c["q"].shape[-3]
    for x, dy in zip("qk", grads):
        total = bound = 0.0
        for a in range(0, n, 2048):
            part = _tokens(c, slice(a, min(n, a + 2048)))
            v = part[x].double().reshape(-1, *part[x].shape[-2:])
            pos = part["positions"].reshape(-1, len(v))
            axes = c["axes"].long().clamp(0, len(pos) - 1) if c["axes"] is not None else torch.zeros_like(c["inv_freq"]).long()
            theta = pos[axes].T.double() * c["inv_freq"].double()
            i, j = (torch.from_numpy(t).to(v.device) for t in ref.pairs(2 * theta.shape[1], interleaved))
            cos, sin = theta.cos()[:, None], theta.sin()[:, None]
            d = dy[..., a:a + 2048, :, :].double().reshape(v.shape)
            g, size = d.clone(), d.abs()
            g[..., i], g[..., j] = d[..., i] * cos + d[..., j] * sin, d[..., j] * cos - d[..., i] * sin
            size[..., i] = size[..., j] = d[..., i].abs() + d[..., j].abs()
            u = v / ((v * v).mean(dim=-1, keepdim=True) + 1e-6).sqrt()
            total = total + (g * u).sum(dim=(0, 1))
            bound = bound + 2.0 ** -17 * (size * u.abs()).sum(dim=(0, 1))
        out += [total, bound]
    return out


@pytest.mark.parametrize("lead,Hq,Hkv,D,R,axes,interleaved,weights", CASES, ids=IDS)
def test_backward(cuda, lead, Hq, Hkv, D, R, axes, interleaved, weights):
    """Of a weight's gradient an fp32 sum has up to 42 rows of a lane, its 8 groups, 4 waves, 12 workgroups of a thread and
    their tree: some 70 additions, 2^-17.8 of the sum of magnitudes, within the reference's 2^-17."""
    import torch
    import cuda_llm_ops_amd as fg
    print(lead, Hq, Hkv, D, R, axes, interleaved, weights, flush=True)
    n = lead[-1]
    c = _make(torch, cuda, lead, Hq, Hkv, D, R, axes=axes, weights=weights)
    gq, gk = (torch.randn(*lead, h, D, device=cuda).to(torch.bfloat16) for h in (Hq, Hkv))
    grads = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    again = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))
    at = _slices(n)
    parts = [fg.qk_norm_rope_backward(gq[..., s, :, :], gk[..., s, :, :], **_tokens(c, s), interleaved=interleaved) for s in at]
    for i in range(2):
        assert _same(torch, grads[i], [p[i] for p in parts], at)
    some = torch.tensor([0, 1, n // 2 + 2, n // 2 + 3, n - 2, n - 1] + list(range(5, n, n // 50)), device=cuda)
    few = dict(_tokens(c, some))
    rows = [grads[0][..., some, :, :], grads[1][..., some, :, :]]
    dws = fg.qk_norm_rope_backward(gq[..., some, :, :], gk[..., some, :, :], **few, interleaved=interleaved)[2:]
    _check_backward(few, gq[..., some, :, :], gk[..., some, :, :], rows + list(dws), interleaved=interleaved)
    if weights is None:
        assert grads[2] is None and grads[3] is None
        return
    want_q, bound_q, want_k, bound_k = _weight_sums(torch, c, (gq, gk), interleaved)
    assert bool(((grads[2].double() - want_q).abs() <= bound_q).all())
    assert bool(((grads[3].double() - want_k).abs() <= bound_k).all())
