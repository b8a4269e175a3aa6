"""Per-head RMSNorm with rotation on the GPU, forward and gradient, against the
formula in 64 bits.

Bounds.  The result is rounded to bf16 once: half a step, 2^-8 of the value.
Before that everything is fp32: the inverse RMS (a sum of D squares, a square
root, a division), three products and a sum err by less than 16 roundings of
2^-24 of the terms, 2^-20 of |a| + |b| for a rotated pair (a, b); the gradient
goes through one more such sum, 2^-18 of the sum of its terms' magnitudes.
"""

import pytest
import torch

from multics_amd.kernels import (qk_head_prologue, qk_head_prologue_backward,
                                 qk_head_prologue_train)
from multics_amd.module import SelfAttention, rope_apply
from tests.gpu_util import need_gpu, say

pytestmark = pytest.mark.gpu
EPS = 1e-6
STEP, F32 = 2.0 ** -8, 2.0 ** -20

CASES = [
    # S, Hq, Hk, D, fused projection, gain dtype, layout
    (1, 1, 1, 128, False, torch.float32, "shd"),
    (1, 24, 24, 128, False, torch.bfloat16, "hsd"),
    (2, 7, 1, 64, True, torch.float32, "shd"),
    (37, 25, 25, 128, False, torch.bfloat16, "hsd"),    # one head past a wave's groups
    (131, 49, 7, 64, True, torch.float32, "hsd"),
    (513, 20, 5, 64, False, torch.bfloat16, "shd"),
    (1999, 12, 2, 128, True, torch.float32, "shd"),
]


def _inputs(S, Hq, Hk, D, fused, gain, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rows = (rnd(S, (Hq + 2 * Hk) * D) * torch.exp(rnd(S, 1))).to(torch.bfloat16)
    qx, kx = rows[:, :Hq * D], rows[:, Hq * D:(Hq + Hk) * D]
    if not fused:
        qx, kx = qx.contiguous(), kx.contiguous()
    angle = rnd(S, D // 2) * 3
    kw = dict(norm_q_w=(1 + 0.3 * rnd(D)).to(gain), norm_k_w=(1 + 0.3 * rnd(D)).to(gain),
              rope_cos=torch.cos(angle), rope_sin=torch.sin(angle), num_heads=Hq, num_kv_heads=Hk,
              eps=EPS)
    dq, dk = rnd(S, Hq, D).to(torch.bfloat16), rnd(S, Hk, D).to(torch.bfloat16)
    return qx, kx, kw, dq, dk


def _formula(x, w, cos, sin, H):
    """(y, |a| + |b| of each element's pair) in 64 bits."""
    S, D = x.shape[0], x.shape[1] // H
    h = x.double().reshape(S, H, D)
    n = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w.double()
    z = torch.view_as_complex(n.reshape(S, H, D // 2, 2).contiguous()) * \
        torch.complex(cos.double(), sin.double())[:, None]
    size = n.abs().reshape(S, H, D // 2, 2).sum(-1, keepdim=True).expand(-1, -1, -1, 2)
    return torch.view_as_real(z).flatten(-2), size.reshape(S, H, D)


@pytest.mark.parametrize("S,Hq,Hk,D,fused,gain,layout", CASES)
def test_forward_matches_the_formula(S, Hq, Hk, D, fused, gain, layout):
    need_gpu()
    qx, kx, kw, _, _ = _inputs(S, Hq, Hk, D, fused, gain)
    say("head norm", S, Hq, Hk, D, fused, gain, layout)
    q, k = qk_head_prologue(qx, kx, out_layout=layout, **kw)
    torch.cuda.synchronize()
    for got, x, w, H in ((q, qx, kw["norm_q_w"], Hq), (k, kx, kw["norm_k_w"], Hk)):
        ref, size = _formula(x, w, kw["rope_cos"], kw["rope_sin"], H)
        assert got.shape == (S, H, D) and got.dtype == torch.bfloat16
        off = (got.double() - ref).abs()
        assert bool((off <= STEP * ref.abs() + 2 * F32 * size).all()), float((off / size).max())


def _grad_formula(x, dy, w, cos, sin, H):
    """(dx, bound of its fp32 error, dw, sum of |terms| of dw) in 64 bits."""
    S, D = x.shape[0], x.shape[1] // H
    h = x.double().reshape(S, H, D)
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    z = torch.view_as_complex(dy.double().reshape(S, H, D // 2, 2).contiguous()) * \
        torch.complex(cos.double(), -sin.double())[:, None]
    dn = torch.view_as_real(z).flatten(-2)
    big = dy.double().abs().reshape(S, H, D // 2, 2).sum(-1, keepdim=True).expand(
        -1, -1, -1, 2).reshape(S, H, D)                      # bounds |dn| and its terms
    xh, dh = h * r, dn * w.double()
    dx = r * (dh - xh * (dh * xh).mean(-1, keepdim=True))
    bh = big * w.double().abs()
    size = r * (bh + xh.abs() * (bh * xh.abs()).mean(-1, keepdim=True))
    return dx, 2.0 ** -18 * size, (dn * xh).sum((0, 1)), (big * xh.abs()).sum((0, 1))


@pytest.mark.parametrize("S,Hq,Hk,D,fused,gain,layout", CASES)
def test_gradient_matches_the_formula(S, Hq, Hk, D, fused, gain, layout):
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(S, Hq, Hk, D, fused, gain)
    if layout == "hsd":         # gradients of head-major storage
        dq, dk = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (dq, dk))
    say("head norm gradient", S, Hq, Hk, D, fused, gain, layout)
    got = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    again = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for x, dy, w, H, dx, dw in ((qx, dq, kw["norm_q_w"], Hq, got[0], got[2]),
                                (kx, dk, kw["norm_k_w"], Hk, got[1], got[3])):
        ref, slack, rw, terms = _grad_formula(x, dy, w, kw["rope_cos"], kw["rope_sin"], H)
        assert dx.shape == x.shape
        off = (dx.double().reshape(ref.shape) - ref).abs()
        assert bool((off <= STEP * (ref.abs() + slack) + slack).all()), float((off / slack).max())
        # fp32 sums of fewer than 256 terms in a row at these sizes, each term
        # itself within 2^-20: 2^-15 of the terms' magnitudes
        assert dw.dtype == torch.float32
        assert bool(((dw.double() - rw).abs() <= 2.0 ** -15 * terms).all())


def test_gradient_matches_differences():
    """Along a random direction, against the 64-bit formula's central difference."""
    need_gpu()
    S, Hq, Hk, D = 33, 6, 3, 64
    qx, kx, kw, dq, dk = _inputs(S, Hq, Hk, D, False, torch.float32, seed=4)
    got = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    g = torch.Generator(device="cuda").manual_seed(9)
    for x, dy, w, H, dx, dw in ((qx, dq, kw["norm_q_w"], Hq, got[0], got[2]),
                                (kx, dk, kw["norm_k_w"], Hk, got[1], got[3])):
        u = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
        uw = torch.randn(D, generator=g, device="cuda", dtype=torch.float64)
        loss = lambda t: (_formula(x.double() + t * u, w.double() + t * uw,  # noqa: E731
                                   kw["rope_cos"], kw["rope_sin"], H)[0] * dy.double()).sum()
        h = 1e-5
        slope = (loss(h) - loss(-h)) / (2 * h)
        mine = (dx.double() * u).sum() + (dw.double() * uw).sum()
        _, slack, _, terms = _grad_formula(x, dy, w, kw["rope_cos"], kw["rope_sin"], H)
        bound = ((STEP * dx.double().abs() + 2 * slack.reshape(dx.shape)) * u.abs()).sum() + \
            (2.0 ** -15 * terms * uw.abs()).sum() + 1e-7 * slope.abs()
        assert (slope - mine).abs() <= bound


def test_autograd_and_module_gradients():
    """The training entry gives the raw gradient, for strided columns too, and
    SelfAttention(qk_norm="head") reaches it: its q and k equal the torch tail
    (which rounds after the norm, the gain and the rotation: three roundings)."""
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(45, 8, 2, 64, True, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (qx, kx, kw["norm_q_w"], kw["norm_k_w"])]
    q, k = qk_head_prologue_train(leaves[0], leaves[1], **{**kw, "norm_q_w": leaves[2],
                                                           "norm_k_w": leaves[3]})
    got = torch.autograd.grad([q, k], leaves, [dq, dk])
    want = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(got[2], want[2].bfloat16()) and torch.equal(got[3], want[3].bfloat16())
    with pytest.raises(RuntimeError, match="qk_head_prologue_train"):
        qk_head_prologue(leaves[0], leaves[1], **kw)

    torch.manual_seed(0)
    m = SelfAttention(320, 5, qk_norm="head").to("cuda", torch.bfloat16)     # dim not k * 512
    m.enable_camera_pose_qk(12, dropout_p=0.0)
    torch.nn.init.normal_(m.cam_q.weight, std=0.1)
    torch.nn.init.normal_(m.norm_q.weight, mean=1.0, std=0.2)
    assert m.norm_q.weight.shape == (64,)
    x = torch.randn(1, 70, 320, device="cuda").to(torch.bfloat16).requires_grad_()
    cam = torch.randn(1, 70, 12, device="cuda").to(torch.bfloat16)
    freqs = torch.polar(torch.ones(70, 1, 32, dtype=torch.float64, device="cuda"),
                        torch.rand(70, 1, 32, dtype=torch.float64, device="cuda"))
    q, k, v = m._project_train(x, freqs, cam)
    pq, pk, pv = (t.view(70, 5, 64) for t in m._project_self_attn_qkv(x, freqs, cam))
    for a, b in ((q, pq), (k, pk)):
        # three roundings against one, and the rotation mixes a pair's
        pair = b.double().reshape(70, 5, 32, 2).abs().sum(-1, keepdim=True).expand(
            -1, -1, -1, 2).reshape(b.shape)
        assert bool(((a.double() - b.double()).abs() <= 4 * STEP * 1.5 * pair).all())
    assert torch.equal(v, pv)
    (q.float().square().sum() + k.float().sum()).backward()
    for p in (x, m.q.weight, m.k.weight, m.norm_q.weight, m.norm_k.weight, m.cam_q.weight):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and bool((p.grad != 0).any())
    with torch.no_grad():
        fq, fk, _ = m._qkv_blocks(x, freqs, cam)
    assert torch.equal(fq, q) and torch.equal(fk, k)


def test_values_that_are_not_finite_stay_in_their_head():
    need_gpu()
    qx, kx, kw, _, _ = _inputs(9, 4, 4, 64, False, torch.float32)
    ref = qk_head_prologue(qx, kx, **kw)
    bad = qx.clone()
    bad[3, 64 + 5] = float("nan")
    bad[5, 130] = float("inf")
    q, k = qk_head_prologue(bad, kx, **kw)
    keep = torch.ones(9, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = keep[5, 2] = False
    assert torch.equal(q[keep], ref[0][keep]) and torch.equal(k, ref[1])
    assert bool(torch.isnan(q[3, 1]).all()) and bool(torch.isnan(q[5, 2, 2:4]).any())
    zero = qk_head_prologue(torch.zeros_like(qx), kx, **kw)[0]
    assert torch.count_nonzero(zero) == 0


def test_more_than_2_31_elements():
    """The last tokens of a long sequence, forward and gradient, equal those of
    the same tokens alone (the gains' gradients are sums over all: not compared)."""
    need_gpu()
    S, H, D, last = 2 ** 31 // (24 * 128) + 100, 24, 128, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    some = torch.randn(997, H * D, generator=g, device="cuda").to(torch.bfloat16)
    qx = some.repeat(-(-S // 997), 1)[:S]
    kx = qx[:, :D].contiguous()
    angle = torch.rand(S, D // 2, generator=g, device="cuda")
    cs, sn = angle.cos(), angle.sin()
    w = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    kw = dict(norm_q_w=w, norm_k_w=w, num_heads=H, num_kv_heads=1, eps=1e-6)
    end = lambda t: t[-last:]  # noqa: E731
    tail = dict(kw, rope_cos=end(cs), rope_sin=end(sn))
    full = dict(kw, rope_cos=cs, rope_sin=sn)
    q, k = qk_head_prologue(qx, kx, **full)
    q2, k2 = qk_head_prologue(end(qx), end(kx), **tail)
    assert torch.equal(end(q), q2) and torch.equal(end(k), k2)
    del q, k
    dq, dk = qx.view(S, H, D), kx.view(S, 1, D)
    got = qk_head_prologue_backward(dq, dk, qx, kx, **full)
    want = qk_head_prologue_backward(end(dq), end(dk), end(qx), end(kx), **tail)
    assert torch.equal(end(got[0]), want[0]) and torch.equal(end(got[1]), want[1])


def test_captured_on_a_side_stream():
    """Forward and gradient recorded into a graph, replayed on new inputs."""
    need_gpu()
    args = [_inputs(77, 6, 2, 128, False, torch.float32, seed=i) for i in range(3)]
    qx, kx, kw, dq, dk = (t.clone() if torch.is_tensor(t) else t for t in args[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        qk_head_prologue(qx, kx, **kw)
        qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_head_prologue(qx, kx, **kw) + qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    for new in args + args:
        for to, t in zip((qx, kx, dq, dk), (new[0], new[1], new[3], new[4])):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = qk_head_prologue(qx, kx, **kw) + qk_head_prologue_backward(dq, dk, qx, kx, **kw)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_training_step_captured():
    """Forward and ``backward()`` of the differentiable form in one graph, the
    warm-up's graphs gone before: replayed gradients equal the eager ones."""
    need_gpu()
    args = [_inputs(61, 4, 2, 64, False, torch.float32, seed=i) for i in range(3)]
    qx, kx, kw, dq, dk = (t.clone() if torch.is_tensor(t) else dict(t) for t in args[0])
    leaves = [t.requires_grad_() for t in (qx, kx, kw["norm_q_w"].clone(), kw["norm_k_w"].clone())]
    kw["norm_q_w"], kw["norm_k_w"] = leaves[2:]

    def step():
        q, k = qk_head_prologue_train(qx, kx, **kw)
        torch.autograd.backward((q, k), (dq, dk))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            for t in leaves:
                t.grad = None
            step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for t in leaves:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    say("capture of a training step")
    with torch.cuda.graph(graph, stream=stream):
        step()
    for new in args + args:
        with torch.no_grad():
            for to, t in zip((qx, kx, dq, dk), (new[0], new[1], new[3], new[4])):
                to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            want = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_one_row_with_a_stride_of_no_meaning():
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(1, 3, 1, 64, False, torch.float32)
    want = qk_head_prologue(qx, kx, **kw) + qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    odd, one = qx.as_strided((1, 192), (1, 1)), kx.as_strided((1, 64), (7, 1))
    got = qk_head_prologue(odd, one, **kw) + qk_head_prologue_backward(
        dq.as_strided((1, 3, 64), (3, 64, 1)), dk.as_strided((1, 1, 64), (1, 5, 1)), odd, one, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_and_empty():
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(8, 4, 2, 64, False, torch.float32)
    bad = [
        (ValueError, dict(num_heads=3)), (ValueError, dict(num_kv_heads=4)),
        (ValueError, dict(num_heads=0)), (NotImplementedError, dict(num_heads=8, num_kv_heads=4)),
        (ValueError, dict(norm_q_w=kw["norm_q_w"][:32])),
        (ValueError, dict(norm_q_w=kw["norm_q_w"].half())),
        (ValueError, dict(rope_cos=kw["rope_cos"][:7])),
        (ValueError, dict(rope_sin=kw["rope_sin"].cpu())), (ValueError, dict(out_layout="sdh")),
    ]
    for exc, change in bad:
        with pytest.raises(exc):
            qk_head_prologue(qx, kx, **{**kw, **change})
    with pytest.raises(NotImplementedError):
        qk_head_prologue(qx.float(), kx, **kw)
    with pytest.raises(ValueError):
        qk_head_prologue(qx, kx[:7], **kw)
    with pytest.raises(ValueError):
        qk_head_prologue_backward(dq[:, :3], dk, qx, kx, **kw)
    with pytest.raises(ValueError):
        qk_head_prologue_backward(dq.float(), dk, qx, kx, **kw)
    none = {**kw, "rope_cos": kw["rope_cos"][:0], "rope_sin": kw["rope_sin"][:0]}
    q, k = qk_head_prologue(qx[:0], kx[:0], **none)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    grads = qk_head_prologue_backward(dq[:0], dk[:0], qx[:0], kx[:0], **none)
    assert grads[0].shape == (0, 256) and torch.count_nonzero(grads[2]) == 0


def _check_gradient(qx, kx, kw, dq, dk, Hq, Hk):
    """The entry's gradient within the bounds of the head of this file."""
    got = qk_head_prologue_backward(dq, dk, qx, kx, **kw)
    for x, dy, w, H, dx, dw in ((qx, dq, kw["norm_q_w"], Hq, got[0], got[2]),
                                (kx, dk, kw["norm_k_w"], Hk, got[1], got[3])):
        ref, slack, rw, terms = _grad_formula(x, dy, w, kw["rope_cos"], kw["rope_sin"], H)
        off = (dx.double().reshape(ref.shape) - ref).abs()
        assert bool((off <= STEP * (ref.abs() + slack) + slack).all()), float((off / slack).max())
        assert bool(((dw.double() - rw).abs() <= 2.0 ** -15 * terms).all())


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (5, 2), (7, 5), (12, 3), (24, 24)])
@pytest.mark.parametrize("D", [64, 128])
def test_gradient_without_an_eps(D, Hq, Hk, monkeypatch):
    """eps = 0, with head counts that leave lanes of a wave without a head."""
    need_gpu()
    monkeypatch.setitem(globals(), "EPS", 0.0)
    qx, kx, kw, dq, dk = _inputs(19, Hq, Hk, D, False, torch.float32)
    assert kw["eps"] == 0.0
    say("head norm gradient, eps 0", D, Hq, Hk)
    _check_gradient(qx, kx, kw, dq, dk, Hq, Hk)


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf"), 1e300])
def test_an_eps_below_0_is_refused(eps):
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(3, 2, 1, 64, False, torch.float32)
    for call in (lambda kw: qk_head_prologue(qx, kx, **kw),
                 lambda kw: qk_head_prologue_train(qx, kx, **kw),
                 lambda kw: qk_head_prologue_backward(dq, dk, qx, kx, **kw)):
        with pytest.raises(ValueError, match="eps"):
            call({**kw, "eps": eps})


@pytest.mark.parametrize("q_gain,k_gain", [(torch.float32, torch.float32),
                                           (torch.bfloat16, torch.float32)])
def test_module_with_fp32_gains_runs_the_pass(q_gain, k_gain, monkeypatch):
    """A bf16 module whose norms are kept in fp32 (or one of them): q and k come
    from the HIP pass with and without autograd, once rounded from the formula."""
    need_gpu()
    from multics_amd import module as mod
    calls = []
    for name in ("qk_head_prologue", "qk_head_prologue_train"):
        fn = getattr(mod, name)
        monkeypatch.setattr(mod, name, lambda *a, fn=fn, name=name, **kw: calls.append(name) or fn(*a, **kw))
    torch.manual_seed(3)
    S, H, D = 41, 3, 64
    m = SelfAttention(H * D, H, qk_norm="head").to("cuda", torch.bfloat16)
    m.norm_q.to(q_gain), m.norm_k.to(k_gain)
    for norm in (m.norm_q, m.norm_k):
        torch.nn.init.normal_(norm.weight, mean=1.0, std=0.2)
    x = torch.randn(1, S, H * D, device="cuda").to(torch.bfloat16)
    angle = torch.rand(S, 1, D // 2, dtype=torch.float64, device="cuda").float().double()
    freqs = torch.polar(torch.ones_like(angle), angle)
    q, k, _ = m._project_train(x, freqs, None)
    torch.autograd.backward((q, k), (torch.ones_like(q), torch.ones_like(k)))
    with torch.no_grad():
        fq, fk, _ = m._qkv_blocks(x, freqs, None)
        assert calls == ["qk_head_prologue_train", "qk_head_prologue"]
        assert torch.equal(fq, q) and torch.equal(fk, k)
        cs, sn = freqs.real[:, 0].float(), freqs.imag[:, 0].float()
        for got, lin, norm in ((q, m.q, m.norm_q), (k, m.k, m.norm_k)):
            assert norm.weight.grad.dtype == norm.weight.dtype
            ref, size = _formula(lin(x)[0], norm.weight, cs, sn, H)
            assert bool(((got.double() - ref).abs() <= STEP * ref.abs() + 2 * F32 * size).all())


def test_gain_sums_of_many_tokens():
    """More tokens than eight for each of the 1,024 workgroups, unequal head counts.
    A sum is fewer than 256 additions in a row here too (k: 16 tokens a wave, three
    steps over the lanes, four waves, 10 rows a thread, 16 threads)."""
    need_gpu()
    qx, kx, kw, dq, dk = _inputs(9001, 12, 2, 64, False, torch.float32, seed=8)
    _check_gradient(qx, kx, kw, dq, dk, 12, 2)


@pytest.mark.parametrize("gain", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cam_dim", [0, 12])
def test_module_gradients_match_64_bits(cam_dim, gain):
    """Gradients of a training projection -- the input, the q and k products, the
    camera adapters and the gains -- against autograd in 64 bits through the same
    module, its q and k rows those that bf16 products gave.

    Bounds: a gradient of a q row is the kernel's (the bounds above, d below); a
    product with it sums d times the other factor, fp32 sums of fewer than 2^9
    terms (2^-15 of the terms), rounded to bf16; x gathers two such products and
    their rounded sum."""
    need_gpu()
    torch.manual_seed(1)
    S, H, D = 70, 5, 64
    m = SelfAttention(H * D, H, qk_norm="head").to("cuda", torch.bfloat16)
    m.norm_q.to(gain), m.norm_k.to(gain)
    for norm in (m.norm_q, m.norm_k):
        torch.nn.init.normal_(norm.weight, mean=1.0, std=0.2)
    x = torch.randn(1, S, H * D, device="cuda").to(torch.bfloat16).requires_grad_()
    cam, adapters = None, [None, None]
    if cam_dim:
        m.enable_camera_pose_qk(cam_dim, dropout_p=0.0)
        adapters = [m.cam_q, m.cam_k]
        for a in adapters:
            torch.nn.init.normal_(a.weight, std=0.1)
        cam = torch.randn(1, S, cam_dim, device="cuda").to(torch.bfloat16)
    angle = torch.rand(S, 1, D // 2, dtype=torch.float64, device="cuda")
    freqs = torch.polar(torch.ones_like(angle), angle)
    grads = [torch.randn(S, H, D, device="cuda").to(torch.bfloat16) for _ in range(2)]
    q, k, _ = m._project_train(x, freqs, cam)
    torch.autograd.backward((q, k), grads)
    with torch.no_grad():
        rows = m._apply_camera_qk(m.q(x), m.k(x), cam)
    cs, sn = freqs.real[:, 0].float(), freqs.imag[:, 0].float()
    xw = x.detach().double()[0]
    want_x, room_x = [], []
    near = lambda got, ref, room: bool(  # noqa: E731
        ((got.double() - ref).abs() <= STEP * (ref.abs() + room) + room).all())
    for row, dy, lin, norm, adapter in zip(rows, grads, (m.q, m.k), (m.norm_q, m.norm_k), adapters):
        row64 = row[0].double().requires_grad_()
        w64 = norm.weight.detach().double().requires_grad_()
        y, _ = _formula(row64, w64, cs, sn, H)
        drow, dw = torch.autograd.grad(y, (row64, w64), dy.double())
        _, slack, _, terms = _grad_formula(row[0], dy, norm.weight.detach(), cs, sn, H)
        slack = slack.reshape(drow.shape)
        d = STEP * (drow.abs() + slack) + slack            # of a row's gradient
        for name, got, other in (("weight", lin.weight, xw), ("bias", lin.bias, torch.ones_like(xw[:, :1])),
                                 ("camera", None if adapter is None else adapter.weight,
                                  None if cam is None else cam[0].double())):
            if got is None:
                continue
            ref = (drow.t() @ other).reshape(got.shape)
            room = ((d + 2.0 ** -15 * drow.abs()).t() @ other.abs()).reshape(got.shape)
            assert near(got.grad, ref, room), name
        w = lin.weight.detach().double()
        want_x.append(drow @ w)
        room = (d + 2.0 ** -15 * drow.abs()) @ w.abs()
        room_x.append(STEP * (want_x[-1].abs() + room) + room)
        assert bool(((norm.weight.grad.double() - dw).abs() <=
                     STEP * dw.abs() + (1 + STEP) * 2.0 ** -15 * terms).all())
    assert near(x.grad[0], sum(want_x), sum(room_x))
