"""Norm and rotation of queries and keys on the GPU against float64 (tests/_rope_reference.py,
which derives the bounds): a bf16 output is off by its rounding, 2^-8 of its value, and
the fp32 steps before it."""
import numpy as np
import pytest

from tests import _rope_reference as ref

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().double().cpu().numpy()


def _make(torch, dev, lead, Hq, Hkv, D, R, seed=1, axes=None, weights="bf16", fused=True, pos="int64", far=0):
    """Inputs of a call; axes: None or the number of them."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    bf = torch.bfloat16
    if fused:
        qkv = torch.randn(*lead, Hq + 2 * Hkv, D, generator=g).to(bf).to(dev)
        q, k = qkv[..., :Hq, :], qkv[..., Hq:Hq + Hkv, :]
    else:
        q, k = (torch.randn(*lead, h, D, generator=g).to(bf).to(dev) for h in (Hq, Hkv))
    c = dict(q=q, k=k)
    c["inv_freq"] = (1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))).float().to(dev)
    n = (axes,) if axes else ()
    c["positions"] = (torch.randint(0, 300, n + tuple(lead), generator=g) + far).to(getattr(torch, pos)).to(dev)
    c["axes"] = torch.randint(0, axes, (R // 2,), generator=g).to(torch.int32).to(dev) if axes else None
    for w in ("q_weight", "k_weight"):
        c[w] = None if weights is None else (1 + 0.3 * torch.randn(D, generator=g)).to(
            bf if weights == "bf16" else torch.float32).to(dev)
    return c


def _theta(c, T):
    if c["positions"] is None:
        return np.zeros((T, 0))
    pos = c["positions"].cpu().numpy()
    pos = pos.reshape(-1, T) if pos.size % T == 0 and pos.size >= T else np.broadcast_to(pos, c["q"].shape[:-2]).reshape(1, T)
    return ref.angles(pos, c["inv_freq"].cpu().numpy(), None if c["axes"] is None else c["axes"].cpu().numpy())


def _within(got, want, bound, what):
    d = np.abs(_np(got).reshape(want.shape) - want)
    assert np.isfinite(d).all(), what
    worst = (d - bound).max() if d.size else 0.0
    assert worst <= 0, (what, worst, d.max())


def _check_forward(c, outs, eps=1e-6, interleaved=False):
    for n, out in zip("qk", outs):
        H, D = c[n].shape[-2:]
        x = _np(c[n]).reshape(-1, H, D)
        w = None if c[n + "_weight"] is None else _np(c[n + "_weight"])
        want, bound = ref.forward(x, w, _theta(c, len(x)), eps, interleaved)
        _within(out, want, 2.0 ** -8 * np.abs(want) + bound * 1.01, n)


def _check_backward(c, gq, gk, outs, eps=1e-6, interleaved=False):
    for n, dy, out, dw in zip("qk", (gq, gk), outs[:2], outs[2:]):
        H, D = c[n].shape[-2:]
        x, dy = _np(c[n]).reshape(-1, H, D), _np(dy).reshape(-1, H, D)
        w = None if c[n + "_weight"] is None else _np(c[n + "_weight"])
        want, bound, want_w, bound_w = ref.backward(dy, x, w, _theta(c, len(x)), eps, interleaved)
        _within(out, want, 2.0 ** -8 * np.abs(want) + bound * 1.01, n)
        if w is None:
            assert dw is None
        else:
            _within(dw, want_w, bound_w, n + "_weight")


CASES = [
    # lead, Hq, Hkv, D, R, axes, interleaved, weights
    ((1, 1), 1, 1, 128, 128, None, False, "bf16"),
    ((3,), 16, 2, 128, 128, None, False, "bf16"),
    ((64,), 64, 8, 128, 128, None, False, "bf16"),
    ((2, 37), 28, 4, 128, 128, 3, False, "bf16"),
    ((2, 37), 28, 4, 128, 128, 3, True, "fp32"),
    ((1, 130), 5, 3, 128, 64, None, False, "bf16"),
    ((1, 130), 5, 3, 128, 64, 2, True, "bf16"),
    ((2, 65), 8, 8, 64, 64, None, False, "fp32"),
    ((2, 65), 7, 1, 64, 16, None, True, "bf16"),
    ((1, 99), 16, 1, 80, 80, None, False, "bf16"),
    ((1, 99), 9, 2, 80, 48, 3, True, "bf16"),
    ((1, 77), 6, 2, 96, 96, None, False, "bf16"),
    ((1, 77), 6, 2, 192, 192, None, True, "bf16"),
    ((1, 77), 6, 2, 176, 112, 4, False, "bf16"),
    ((2, 33), 3, 5, 256, 256, None, False, "fp32"),
    ((2, 33), 3, 5, 240, 16, None, True, "bf16"),
    ((1, 41), 4, 2, 16, 16, None, False, "bf16"),
    ((1, 41), 4, 2, 32, 32, None, False, None),
    ((2, 300), 32, 8, 128, 128, 3, True, None),
    ((2, 600), 32, 8, 128, 128, None, False, "bf16"),
    ((3, 171), 128, 8, 64, 64, None, False, "bf16"),
    ((1, 1500), 17, 3, 128, 128, 3, False, "bf16"),
]


@pytest.mark.parametrize("lead,Hq,Hkv,D,R,axes,interleaved,weights", CASES)
def test_forward_and_backward(cuda, lead, Hq, Hkv, D, R, axes, interleaved, weights):
    import torch
    import cuda_llm_ops_amd as fg
    print(lead, Hq, Hkv, D, R, axes, interleaved, weights, flush=True)
    c = _make(torch, cuda, lead, Hq, Hkv, D, R, axes=axes, weights=weights)
    outs = fg.qk_norm_rope(**c, interleaved=interleaved)
    assert outs[0].is_contiguous() and outs[1].is_contiguous()
    _check_forward(c, outs, interleaved=interleaved)
    gq, gk = torch.randn_like(outs[0]), torch.randn_like(outs[1])
    grads = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    _check_backward(c, gq, gk, grads, interleaved=interleaved)
    again = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("lead,Hq,Hkv,D,R,axes,interleaved,weights", [
    ((2, 4501), 16, 8, 128, 128, 3, True, "bf16"),
    ((1, 10007), 17, 3, 128, 96, None, False, "fp32"),
    ((1, 4500), 9, 2, 256, 256, None, False, "bf16"),
    ((20000,), 4, 2, 64, 64, None, True, "bf16"),
])
def test_many_rows(cuda, lead, Hq, Hkv, D, R, axes, interleaved, weights):
    """Items of many rows, more than one for each workgroup.  Of a weight's gradient an fp32 sum has up to 24
    rows of a lane, its 8 groups, 4 waves, 12 workgroups of a thread and their tree: some 50 additions, 2^-18.3 of
    the sum of magnitudes, within the reference's 2^-17."""
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, lead, Hq, Hkv, D, R, axes=axes, weights=weights)
    outs = fg.qk_norm_rope(**c, interleaved=interleaved)
    _check_forward(c, outs, interleaved=interleaved)
    gq, gk = torch.randn_like(outs[0]), torch.randn_like(outs[1])
    grads = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    _check_backward(c, gq, gk, grads, interleaved=interleaved)
    again = fg.qk_norm_rope_backward(gq, gk, **c, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_norm_alone(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 9), 4, 2, 128, 128)
    c.update(positions=None, inv_freq=None)
    outs = fg.qk_norm_rope(**c)
    _check_forward(c, outs)
    gq, gk = torch.randn_like(outs[0]), torch.randn_like(outs[1])
    _check_backward(c, gq, gk, fg.qk_norm_rope_backward(gq, gk, **c))


def test_nothing_to_do_is_the_identity(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 9), 4, 2, 128, 128, weights=None)
    c.update(positions=None, inv_freq=None)
    outs = fg.qk_norm_rope(**c)
    assert torch.equal(outs[0], c["q"]) and torch.equal(outs[1], c["k"])


@pytest.mark.parametrize("far,pos", [(32768, "int32"), (1 << 20, "int64"), (-5000, "int32"), ((1 << 31) - 400, "int64")])
def test_far_positions(cuda, far, pos):
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (1, 50), 4, 2, 128, 128, pos=pos, far=far)
    _check_forward(c, fg.qk_norm_rope(**c))
    _check_forward(c, fg.qk_norm_rope(**c, interleaved=True), interleaved=True)


def test_forms_of_positions(cuda):
    """[S] for every batch, expanded and strided ones, and axes out of range."""
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (3, 20), 4, 2, 64, 64, axes=3)
    wide = torch.randint(0, 99, (20, 3, 5, 2), device=cuda)
    c["positions"] = wide[..., 0].permute(2, 1, 0)[:3]
    assert not c["positions"].is_contiguous()
    _check_forward(c, fg.qk_norm_rope(**c))
    c["axes"] = c["axes"] * 5 - 3            # -3, 2, 7: clamped to 0, 2, 2
    _check_forward(c, fg.qk_norm_rope(**c))
    one = torch.arange(20, device=cuda) * 3
    c["axes"] = None
    for p in (one, one.to(torch.int32), one.expand(3, 20), one.expand(1, 3, 20)):
        full = dict(c, positions=one.expand(3, 20).contiguous())
        outs = fg.qk_norm_rope(**dict(c, positions=p))
        _check_forward(full, outs)


def test_in_place_and_given_outputs(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 70), 8, 2, 128, 128)
    want = fg.qk_norm_rope(**c)
    buf = torch.full((2, 70, 11, 128), 7.0, dtype=torch.bfloat16, device=cuda)
    outs = fg.qk_norm_rope(**c, q_out=buf[:, :, :8], k_out=buf[:, :, 9:])
    assert torch.equal(buf[:, :, :8], want[0]) and torch.equal(buf[:, :, 9:], want[1]) and bool((buf[:, :, 8] == 7).all())
    assert outs[0].data_ptr() == buf.data_ptr()
    q, k = c["q"], c["k"]
    v = q._base if q._base is not None else q
    rest = v[:, :, 10:].clone()
    before = q._version
    fg.qk_norm_rope(**c, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v[:, :, 10:], rest)
    assert q._version > before


def test_rows_of_other_strides(cuda):
    """Rows that lie by heads, and rows that are not 16-byte aligned (they are copied)."""
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 30), 8, 2, 128, 128, fused=False)
    want = fg.qk_norm_rope(**c)
    gq, gk = torch.randn_like(c["q"]), torch.randn_like(c["k"])
    grads = fg.qk_norm_rope_backward(gq, gk, **c)

    def by_heads(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):
        out = torch.zeros(t.shape[:-1] + (t.shape[-1] + 3,), dtype=t.dtype, device=t.device)[..., 1:-2]
        out.copy_(t)
        return out

    for f in (by_heads, odd):
        d = dict(c, q=f(c["q"]), k=f(c["k"]))
        assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope(**d), want))
        assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope_backward(f(gq), f(gk), **d), grads))
    d = dict(c, q_weight=c["q_weight"].new_empty(129)[1:].copy_(c["q_weight"]),
             inv_freq=c["inv_freq"].new_empty(65)[1:].copy_(c["inv_freq"]))
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope(**d), want))


def test_offsets_past_32_bits(cuda):
    """Batches and heads more than 2^32 bytes apart, outputs too."""
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (3, 40), 8, 2, 128, 128, fused=False)
    want = fg.qk_norm_rope(**c)
    gq, gk = torch.randn_like(c["q"]), torch.randn_like(c["k"])
    grads = fg.qk_norm_rope_backward(gq, gk, **c)
    far = (1 << 31) + 256   # elements
    room = torch.empty(2 * far + 40 * 8 * 128, dtype=torch.bfloat16, device=cuda)

    def spread(t):
        return room.as_strided(t.shape, (far, t.shape[2] * 128, 128, 1)).copy_(t)

    d = dict(c, q=spread(c["q"]))
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope(**d), want))
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope_backward(gq, gk, **d), grads))
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope_backward(spread(gq), gk, **c), grads))
    out = room.as_strided(c["q"].shape, (far, 8 * 128, 128, 1))
    assert torch.equal(fg.qk_norm_rope(**c, q_out=out)[0], want[0])
    heads = room.as_strided((3, 40, 2, 128), (40 * 128, 128, far, 1)).copy_(c["k"])
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope(**dict(c, k=heads)), want))
    assert all(torch.equal(a, b) for a, b in zip(fg.qk_norm_rope_backward(gq, gk, **dict(c, k=heads)), grads))


def test_empty_and_odd_values(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 0), 8, 2, 128, 128, fused=False)
    outs = fg.qk_norm_rope(**c)
    assert outs[0].shape == (2, 0, 8, 128)
    grads = fg.qk_norm_rope_backward(c["q"], c["k"], **c)
    assert grads[0].shape == (2, 0, 8, 128) and bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())
    # rows of zeros; NaN and infinities stay in their rows
    c = _make(torch, cuda, (1, 40), 8, 2, 128, 64, fused=False)
    clean = fg.qk_norm_rope(**c)
    c["q"][0, 3, 2] = 0
    c["q"][0, 7, 1, 5] = float("nan")
    c["k"][0, 9, 0, 100] = float("inf")
    q, k = fg.qk_norm_rope(**c)
    assert bool((q[0, 3, 2] == 0).all()) and bool(q[0, 7, 1].isnan().all())
    same = torch.ones(40, 8, dtype=torch.bool, device=cuda)
    same[3, 2] = same[7, 1] = False
    assert torch.equal(q[0][same], clean[0][0][same])
    c["k"][0, 9, 0] = c["k"][0, 8, 0]
    # without a norm an infinity that is not rotated stays one, and its neighbours as they were
    c.update(q_weight=None, k_weight=None)
    c["k"][0, 9, 0, 100] = float("inf")
    c["q"][0, 7, 1, 5] = 1.0
    _, k = fg.qk_norm_rope(**c)
    assert bool(k[0, 9, 0, 100].isinf()) and int((~k[0, 9, 0].isfinite()).sum()) == 1
    # eps 0: rows of no token leave nothing behind, a row of zeros is 0 * inf as the formula says
    c = _make(torch, cuda, (1, 3), 3, 1, 128, 128)
    _check_forward(c, fg.qk_norm_rope(**c, eps=0.0), eps=0.0)
    gq, gk = torch.randn_like(c["q"]), torch.randn_like(c["k"])
    _check_backward(c, gq, gk, fg.qk_norm_rope_backward(gq, gk, **c, eps=0.0), eps=0.0)


def test_small_and_large_values(cuda):
    import torch
    import cuda_llm_ops_amd as fg
    for size in (1e-12, 2.0 ** 40):
        c = _make(torch, cuda, (1, 20), 4, 2, 128, 128, fused=False)
        c["q"], c["k"] = c["q"] * size, c["k"] * size
        _check_forward(c, fg.qk_norm_rope(**c))


def test_another_stream_and_graphs(cuda):
    """Calls on a stream of their own, and two captured graphs replayed with eager work between."""
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 90), 8, 2, 128, 128, fused=False)
    gq, gk = torch.randn_like(c["q"]), torch.randn_like(c["k"])
    want, grads = fg.qk_norm_rope(**c), fg.qk_norm_rope_backward(gq, gk, **c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fg.qk_norm_rope(**c) + fg.qk_norm_rope_backward(gq, gk, **c)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want + grads))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fg.qk_norm_rope(**c) + fg.qk_norm_rope_backward(gq, gk, **c)
        graphs.append((graph, out))
    for i in range(4):
        c["q"].mul_(-1.5)
        gk.add_(0.25)
        want = fg.qk_norm_rope(**c) + fg.qk_norm_rope_backward(gq, gk, **c)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_workspace_of_the_c_abi(cuda):
    """The backward's own workspace: too small and misaligned ones are refused, one that is
    large enough gives the same bits as the library's."""
    import ctypes
    import torch
    import cuda_llm_ops_amd as fg
    c = _make(torch, cuda, (2, 50), 8, 2, 128, 128, fused=False, pos="int32")
    gq, gk = torch.randn_like(c["q"]), torch.randn_like(c["k"])
    want = fg.qk_norm_rope_backward(gq, gk, **c)
    a = RopeBackwardArgs()
    f = a.fwd
    f.q, f.k, f.positions, f.inv_freq = (c[n].data_ptr() for n in ("q", "k", "positions", "inv_freq"))
    f.q_weight, f.k_weight, f.weights_bf16 = c["q_weight"].data_ptr(), c["k_weight"].data_ptr(), 1
    f.num_axes, f.batch, f.seqlen, f.num_q_heads, f.num_kv_heads, f.head_dim, f.rotary_dim, f.eps = 1, 2, 50, 8, 2, 128, 128, 1e-6
    f.positions_stride[:] = [0, 50, 1]
    out = [torch.empty_like(t) for t in want]
    a.grad_q_out, a.grad_k_out = gq.data_ptr(), gk.data_ptr()
    a.grad_q, a.grad_k, a.grad_q_weight, a.grad_k_weight = (t.data_ptr() for t in out)
    for st, h in ((f.q_stride, 8), (f.k_stride, 2), (a.grad_q_out_stride, 8), (a.grad_k_out_stride, 2), (a.grad_q_stride, 8),
                  (a.grad_k_stride, 2)):
        st[:] = [50 * h * 128, h * 128, 128]
    L = ctypes.CDLL(fg.LIB_PATH)
    fn = L.fgqa_qk_norm_rope_backward
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    need = ctypes.c_size_t(0)
    assert L.fgqa_qk_norm_rope_backward_workspace_bytes(ctypes.byref(a), ctypes.byref(need)) == 0 and need.value > 0
    stream = torch.cuda.current_stream().cuda_stream
    work = torch.empty(need.value + 256, dtype=torch.uint8, device=cuda)
    a.workspace, a.workspace_bytes = work.data_ptr(), need.value - 1
    assert fn(ctypes.byref(a), stream) == -3
    a.workspace, a.workspace_bytes = work.data_ptr() + 16, need.value
    assert fn(ctypes.byref(a), stream) == -2
    a.workspace, a.workspace_bytes = None, need.value
    assert fn(ctypes.byref(a), stream) == -3
    for ws, n in ((work.data_ptr(), need.value), (None, 0)):
        a.workspace, a.workspace_bytes = ws, n
        for t in out:
            t.fill_(float("nan"))
        assert fn(ctypes.byref(a), stream) == 0
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def _rope_structs():
    import ctypes as C
    three = C.c_int64 * 3

    class Forward(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("q", "k", "q_out", "k_out", "positions", "inv_freq", "axes", "q_weight", "k_weight")] + [
            (n, C.c_int32) for n in ("positions_int64", "weights_bf16", "num_axes", "batch", "seqlen", "num_q_heads",
                                     "num_kv_heads", "head_dim", "rotary_dim", "interleaved")] + [("eps", C.c_float)] + [
            (n, three) for n in ("q_stride", "k_stride", "q_out_stride", "k_out_stride", "positions_stride")]

    class Backward(C.Structure):
        _fields_ = [("fwd", Forward)] + [(n, C.c_void_p) for n in (
            "grad_q_out", "grad_k_out", "grad_q", "grad_k", "grad_q_weight", "grad_k_weight")] + [
            (n, three) for n in ("grad_q_out_stride", "grad_k_out_stride", "grad_q_stride", "grad_k_stride")] + [
            ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]

    return Forward, Backward


RopeArgs, RopeBackwardArgs = _rope_structs()
