"""The norm, the product with its epilogue and the cross attention on the GPU, forward
and gradients, against the formulas in 64 bits.

Bounds.  A result is rounded once to its type: ``STEP``, half a step, 2^-8 of a bf16 value
and 2^-11 of an fp16 one.  Everything before is fp32: a sum of n terms errs by less than
(n + 8) 2^-24 of the terms' magnitudes in any order; exp2, reciprocals and roots by less
than 2^-20 together.  What else is rounded to 16 bits on the way (the values before the
activation that a gradient reads, dz, P, dS) enters with one STEP of it each, through the
slopes of what follows; each bound below adds them up, term by term.
"""

import math

import pytest
import torch

from multics_amd import kernels
from multics_amd.module import CrossAttention, FeedForward, RMSNorm
from tests.gpu_util import need_gpu, say

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
U = 2.0 ** -24


def _step(t):
    return torch.finfo(t).eps / 2


def _rnd(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def _within(got, ref, slack):
    """|got - ref| within a rounding of got's type and ``slack``."""
    assert got.shape == ref.shape, (got.shape, ref.shape)
    off = (got.double() - ref).abs()
    tol = _step(got.dtype) * (ref.abs() + slack) + slack + (2.0 ** -25 if got.dtype == FP16 else 1e-38)
    assert bool((off <= tol).all()), float((off / tol).max())


# ---- norm ------------------------------------------------------------------------------

NORMS = [
    # M, C, type, gain, residual
    (1, 1, BF16, torch.float32, False),
    (2, 1536, BF16, torch.float32, True),
    (5, 77, FP16, FP16, True),              # 2-byte accesses
    (37, 512, BF16, BF16, False),
    (3, 2048, FP16, torch.float32, True),
    (9, 2049, BF16, torch.float32, True),   # four waves a row
    (4, 5120, BF16, BF16, True),
    (3, 8193, BF16, torch.float32, False),  # sixteen
    (2, 16384, FP16, torch.float32, True),
    (2100, 640, BF16, torch.float32, True),  # past the workgroups that sum the gain's gradient
]


def _norm_case(M, C, t, gain, residual, seed=0):
    r = _rnd(seed)
    x = (r(M, C) * torch.exp(r(M, 1))).to(t)
    res = (2 * r(M, C)).to(t) if residual else None
    return x, (1 + 0.3 * r(C)).to(gain), res, r(M, C).to(t), r(M, C).to(t) if residual else None


def _norm_formula(x, w, res, eps=1e-6):
    h = x.double() + (0 if res is None else res.double())
    s = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, s, h * s * w.double()


@pytest.mark.parametrize("M,C,t,gain,residual", NORMS)
def test_norm_matches_the_formula(M, C, t, gain, residual):
    need_gpu()
    x, w, res, dy, dh = _norm_case(M, C, t, gain, residual)
    say("rms norm", M, C, t, gain, residual)
    got = kernels.rms_norm(x, w, eps=1e-6, residual=res)
    h, s, y = _norm_formula(x, w, res)
    if residual:
        _within(got[1], h, U * (x.double().abs() + res.double().abs()))
        got = got[0]
    # h's own rounding to fp32, the mean of C squares, a root, a division, two products
    slack = 2.0 ** -20 * y.abs() + (C + 8) * U * y.abs()
    if residual:
        slack = slack + U * (x.double().abs() + res.double().abs()) * s * w.double().abs()
    _within(got, y, slack)
    say("its gradient")
    dx, dw = kernels.rms_norm_backward(dy, x, w, eps=1e-6, residual=res, dh=dh)
    again = kernels.rms_norm_backward(dy, x, w, eps=1e-6, residual=res, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
    xh, g = h * s, dy.double() * w.double()
    want = s * (g - xh * (g * xh).mean(-1, keepdim=True))
    size = s * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if residual:
        want = want + dh.double()
    # two means of C terms, each entering once or twice
    _within(dx, want, (2.0 ** -19 + 4 * (C + 8) * U) * (size + want.abs()))
    terms = (dy.double() * xh).abs().sum(0)
    assert dw.dtype == torch.float32
    assert bool(((dw.double() - (dy.double() * xh).sum(0)).abs() <=
                 (2.0 ** -20 + (C + M + 16) * U) * terms + 1e-30).all())


def test_norm_under_autograd():
    need_gpu()
    x, w, res, dy, dh = _norm_case(33, 264, BF16, torch.float32, True, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    y, h = kernels.rms_norm_train(leaves[0], leaves[1], eps=1e-6, residual=leaves[2])
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    dx, dw = kernels.rms_norm_backward(dy, x, w, eps=1e-6, residual=res, dh=dh)
    assert all(torch.equal(a, b) for a, b in zip(got, (dx, dw, dx)))
    # one of the outputs alone
    y, h = kernels.rms_norm_train(leaves[0], leaves[1], eps=1e-6, residual=leaves[2])
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert torch.equal(got[0], kernels.rms_norm_backward(dy, x, w, eps=1e-6, residual=res)[0])
    got = torch.autograd.grad(h, leaves, dh)
    assert torch.equal(got[0], dh) and torch.equal(got[2], dh) and not got[1].any()
    with pytest.raises(RuntimeError):
        kernels.rms_norm(leaves[0], w, eps=1e-6)


def test_norm_reads_views():
    """Columns of a wider tensor, expanded and transposed rows, odd strides."""
    need_gpu()
    r = _rnd(5)
    w = 1 + 0.1 * r(64)
    wide = r(40, 200).to(BF16)
    for x in (wide[:, 8:72], wide[:, 3:67], wide[:1, :64].expand(40, 64), wide[:, :64].t().contiguous().t(),
              wide[:, :128].reshape(10, 4, 2, 64), wide[::3, 64:128]):
        say("norm of a view", tuple(x.shape), x.stride())
        dy = torch.ones_like(x)
        y, want = (kernels.rms_norm(t, w, eps=1e-6) for t in (x, x.contiguous()))
        a, b = (kernels.rms_norm_backward(dy, t, w, eps=1e-6) for t in (x, x.contiguous()))
        if x.data_ptr() % 16 == 0:
            assert torch.equal(y, want) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            continue
        # 2-byte accesses deal the channels to other lanes, so the 64 squares of a row add up in
        # another order: either sum errs by (64 + 8) 2^-24 of itself, which may turn a rounding
        # of y or dx (at most a whole step apart) and enters each of dw's 40 terms (here at most
        # |x| / rms <= 8, as sqrt(64) bounds it)
        for got, ref in ((y, want), (a[0], b[0])):
            assert bool(((got.double() - ref.double()).abs() <= 2.0 ** -7 * ref.double().abs() + 2.0 ** -16).all())
        assert bool(((a[1] - b[1]).abs() <= 40 * 8 * 2 * (64 + 40 + 16) * U).all())


# ---- product with its epilogue -----------------------------------------------------------

LINEARS = [
    # M, K, N, activation, gates, residual, type
    (1, 8, 1, None, 0, False, BF16),
    (1, 1536, 200, "gelu_tanh", 0, True, BF16),
    (16, 100, 33, "silu", 1, True, FP16),          # padded channels
    (40, 999, 130, "gelu", 4, True, BF16),
    (64, 520, 257, None, 64, True, BF16),          # a gate for each row
    (65, 64, 64, "silu", 0, False, BF16),          # the first size over tiles
    (127, 72, 9, "gelu_tanh", 0, True, FP16),
    (130, 1000, 255, "gelu", 2, False, BF16),
    (257, 260, 520, "gelu_tanh", 257, True, BF16),
    (300, 2049, 129, None, 3, True, BF16),         # K in parts, a ragged last tile
    (1000, 136, 1032, "gelu_tanh", 5, True, BF16),
    (1, 70, 4099, None, 0, False, FP16),
    (600, 8, 8, "silu", 0, False, BF16),
    (2, 2500, 33, "silu", 2, True, BF16),          # eight rows or fewer: every count of rows, K past
    (3, 4104, 10, "gelu_tanh", 1, True, FP16),     # a pass of the waves, channels past the last group
    (4, 2049, 3, None, 0, True, BF16),
    (5, 512, 1, "gelu", 5, True, FP16),
    (7, 520, 63, "silu", 0, False, BF16),
    (8, 6000, 72, "gelu_tanh", 2, True, BF16),
    (9, 2056, 100, None, 3, True, FP16),
    (16, 4000, 4000, "silu", 4, True, BF16),       # few rows of many weights: over tiles
    (2305, 2400, 8000, "silu", 5, True, BF16),     # the rows of a last round in small tiles, dw's too
    (2305, 520, 7999, "gelu_tanh", 461, True, FP16),
]
LIPSCHITZ = 1.2          # bounds every activation's slope; their second derivatives are under 1


def _linear_case(M, K, N, act, gates, residual, t, seed=0):
    r = _rnd(seed)
    x, w, b = r(M, K).to(t), (r(N, K) / math.sqrt(K)).to(t), (0.3 * r(N)).to(t)
    return x, w, b, (r(M, N).to(t) if residual else None), ((0.6 * r(gates, N)).to(t) if gates else None), \
        r(M, N).to(t)


def _act64(z, act):
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act == "gelu":
        return torch.nn.functional.gelu(z)
    return torch.nn.functional.silu(z) if act == "silu" else z


def _linear_formula(x, w, b, res, gate, act):
    """(z, act(z), y) with z a leaf's, and the fp32 slack of z."""
    x, w, b = x.double(), w.double(), b.double()
    z = x @ w.t() + b
    size = x.abs() @ w.t().abs() + b.abs()
    slack = (x.shape[1] + 8) * U * size
    a = _act64(z, act)
    g = torch.ones_like(z) if gate is None else gate.double().repeat_interleave(z.shape[0] // gate.shape[0], 0)
    y = g * a + (0 if res is None else res.double())
    return z, a, g, y, slack


@pytest.mark.parametrize("M,K,N,act,gates,residual,t", LINEARS)
def test_product_matches_the_formula(M, K, N, act, gates, residual, t):
    need_gpu()
    x, w, b, res, gate, _ = _linear_case(M, K, N, act, gates, residual, t)
    say("linear", M, K, N, act, gates, residual, t)
    got = kernels.linear_act(x, w, b, activation=act, residual=res, gate=gate)
    assert torch.equal(got, kernels.linear_act(x, w, b, activation=act, residual=res, gate=gate))
    z, a, g, y, zs = _linear_formula(x, w, b, res, gate, act)
    slack = g.abs() * (LIPSCHITZ * zs + 2.0 ** -19 * z.abs()) + 4 * U * (y.abs() + (g * a).abs())
    _within(got, y, slack)


@pytest.mark.parametrize("M,K,N,act,gates,residual,t", LINEARS)
def test_product_gradients_match_the_formula(M, K, N, act, gates, residual, t):
    need_gpu()
    x, w, b, res, gate, dy = _linear_case(M, K, N, act, gates, residual, t, seed=1)
    say("linear gradient", M, K, N, act, gates, residual, t)
    names = [n for n, v in (("x", x), ("w", w), ("b", b), ("res", res), ("gate", gate)) if v is not None]
    leaves = {n: v.clone().requires_grad_() for n, v in (("x", x), ("w", w), ("b", b), ("res", res),
                                                        ("gate", gate)) if v is not None}
    y = kernels.linear_act_train(leaves["x"], leaves["w"], leaves["b"], activation=act, residual=leaves.get("res"),
                                 gate=leaves.get("gate"))
    got = dict(zip(names, torch.autograd.grad(y, [leaves[n] for n in names], dy)))
    z, a, g, _, zs = _linear_formula(x, w, b, res, gate, act)
    zl = z.clone().requires_grad_()
    slope, = torch.autograd.grad(_act64(zl, act).sum(), zl)
    step = _step(t)
    # z as kept: rounded once, except where nothing reads it
    dz_in = zs + (step * (z.abs() + zs) + 2.0 ** -25 if act else 0)
    d = dy.double()
    dz = d * g * slope
    e_dz = (d * g).abs() * (dz_in + 2.0 ** -19 * (1 + z.abs()))
    # dz as an operand: rounded once more (not where it is dy itself)
    e_op = e_dz + (step * (dz.abs() + e_dz) + (2.0 ** -25 if t == FP16 else 0) if act or gates else 0)
    X, W = x.double().abs(), w.double().abs()
    A = dz.abs() + e_op
    _within(got["x"], dz @ w.double(), e_op @ W + (N + 8) * U * (A @ W))
    _within(got["w"], dz.t() @ x.double(), e_op.t() @ X + (M + 8) * U * (A.t() @ X))
    _within(got["b"], dz.sum(0), (e_dz + (M + 16) * U * A).sum(0))
    if residual:
        assert torch.equal(got["res"], dy)
    if gates:
        kept = zs + step * (z.abs() + zs) + 2.0 ** -25
        terms = d.abs() * (LIPSCHITZ * kept + 2.0 ** -19 * z.abs() + (M + 16) * U * a.abs())
        _within(got["gate"], (d * a).reshape(gates, M // gates, N).sum(1), terms.reshape(gates, M // gates, N).sum(1))


def test_product_gradient_matches_differences():
    """Along a random direction, against the 64-bit formula's central difference."""
    need_gpu()
    x, w, b, res, gate, dy = _linear_case(48, 72, 40, "gelu_tanh", 3, True, BF16, seed=7)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, gate)]
    y = kernels.linear_act_train(*leaves[:3], activation="gelu_tanh", residual=res, gate=leaves[3])
    got = torch.autograd.grad(y, leaves, dy)
    r, h = _rnd(8), 1e-4
    along = [r(*t.shape).double() for t in leaves]
    f = lambda s: (dy.double() * _linear_formula(*(t.double() + s * d for t, d in zip((x, w, b), along[:3])),  # noqa: E731
                                                 res, gate.double() + s * along[3], "gelu_tanh")[3]).sum()
    want = float((f(h) - f(-h)) / (2 * h))
    have = float(sum((g.double() * d).sum() for g, d in zip(got, along)))
    # each gradient within about three roundings of 2^-8 of its entries, random over the direction;
    # the differences err by h^2 times a third derivative
    size = math.sqrt(sum(float((g.double() * d).square().sum()) for g, d in zip(got, along)))
    assert abs(have - want) <= 6 * 3 * 2.0 ** -8 * size


def test_product_in_place_and_views():
    need_gpu()
    r = _rnd(11)
    x, w, b = r(3, 50, 64).to(BF16), r(72, 64).to(BF16), r(72).to(BF16)
    res = r(3, 50, 72).to(BF16)
    gate = r(3, 5, 72).to(BF16)
    want = kernels.linear_act(x, w, b, activation="silu", residual=res, gate=gate)
    flat = kernels.linear_act(x.reshape(150, 64), w, b, activation="silu", residual=res.reshape(150, 72),
                              gate=gate.reshape(15, 72))
    assert torch.equal(want.reshape(150, 72), flat)
    mine = res.clone()
    assert kernels.linear_act(x, w, b, activation="silu", residual=mine, gate=gate, out=mine) is mine
    assert torch.equal(mine, want)
    # weights and rows inside wider tensors, transposed, at odd addresses
    wide = torch.zeros(72, 200, dtype=BF16, device="cuda")
    wide[:, 8:72] = w
    assert torch.equal(kernels.linear_act(x, wide[:, 8:72], b, activation="silu", residual=res, gate=gate), want)
    wide[:, 3:67] = w
    assert torch.equal(kernels.linear_act(x, wide[:, 3:67], b, activation="silu", residual=res, gate=gate), want)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kernels.linear_act(xt, w.t().contiguous().t(), b, activation="silu", residual=res, gate=gate),
                       want)
    # one gate for all rows, a broadcast residual, no rows
    one = kernels.linear_act(x, w, b, gate=gate[0, 0])
    assert torch.equal(one, kernels.linear_act(x, w, b, gate=gate[:1, :1].expand(3, 1, 72)))
    assert kernels.linear_act(x[:0], w, b).shape == (0, 50, 72)
    assert kernels.linear_act(x[0, 0], w, b).shape == (72,)
    empty = kernels.linear_act_backward(torch.empty(0, 72, dtype=BF16, device="cuda"), x[0, :0], w)
    assert empty["x"].shape == (0, 64) and not empty["weight"].any()


def test_rows_past_the_end_are_left_alone():
    """An output that is the first rows of a larger tensor: nothing behind it changes."""
    need_gpu()
    r = _rnd(13)
    for M, K, N in ((3, 64, 40), (70, 64, 24), (129, 512, 136)):
        buf = torch.full((M + 300, N), 7.0, dtype=BF16, device="cuda")
        kernels.linear_act(r(M, K).to(BF16), r(N, K).to(BF16), out=buf[:M])
        torch.cuda.synchronize()
        assert bool((buf[M:] == 7).all())
    out = torch.full((2, 40, 2, 64), 7.0, dtype=BF16, device="cuda")
    q, k = r(1, 33, 2, 64).to(BF16), r(1, 20, 2, 64).to(BF16)
    kernels.cross_attention(q, k, k, out=out[:1, :33])
    assert bool((out[0, 33:] == 7).all()) and bool((out[1] == 7).all())


def test_values_that_are_not_numbers_stay_in_their_rows():
    need_gpu()
    r = _rnd(17)
    x, w = r(200, 256).to(BF16), r(320, 256).to(BF16)
    clean = kernels.linear_act(x, w, activation="gelu_tanh")
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[77, 5] = bad
        got = kernels.linear_act(y, w, activation="gelu_tanh")
        keep = torch.arange(200, device="cuda") != 77
        assert torch.equal(got[keep], clean[keep]) and not bool(torch.isfinite(got[77]).all())


def test_product_of_many_gates():
    """More gates than a launch has rows of workgroups, each of more rows than one workgroup takes."""
    need_gpu()
    F, per = 65600, 5
    x, w, _, _, gate, dy = _linear_case(F * per, 8, 8, None, F, False, BF16, seed=3)
    z = kernels.linear_act(x, w)
    got = kernels.linear_act_backward(dy, x, w, preact=z, gate=gate, need=("gate",))["gate"]
    ref = (dy.double() * z.double()).view(F, per, 8)
    _within(got, ref.sum(1), (per + 8) * U * ref.abs().sum(1))
    assert torch.equal(kernels.linear_act(x, w, gate=gate)[-per:], kernels.linear_act(x[-per:], w, gate=gate[-1:]))


def test_offsets_past_32_bits():
    """Rows and sums over rows that lie behind the first 4 GiB of their tensors."""
    need_gpu()
    r = _rnd(23)
    tail = 300
    M, C = 1_500_000, 1536
    x = torch.zeros(M, C, dtype=BF16, device="cuda")
    w = 1 + 0.1 * r(C)
    x[-tail:] = r(tail, C).to(BF16)
    assert torch.equal(kernels.rms_norm(x, w, eps=1e-6)[-tail:], kernels.rms_norm(x[-tail:], w, eps=1e-6))
    say("norm past 4 GiB")
    # a product over those rows: x [M, C] as operand, dw a sum over M whose terms lie at its end
    wt, dy = r(72, C).to(BF16), torch.zeros(M, 72, dtype=BF16, device="cuda")
    dy[-tail:] = r(tail, 72).to(BF16)
    y = kernels.linear_act(x, wt)
    say("product past 4 GiB")
    ref = x[-tail:].double() @ wt.double().t()
    _within(y[-tail:], ref, (C + 8) * U * (x[-tail:].double().abs() @ wt.double().abs().t()))
    assert not y[:-tail].any()
    got = kernels.linear_act_backward(dy, x, wt, need=("x", "weight", "bias"))
    say("its gradients past 4 GiB")
    a, b = dy[-tail:].double(), x[-tail:].double()
    _within(got["weight"], a.t() @ b, (M + 8) * U * (a.abs().t() @ b.abs()))
    _within(got["x"][-tail:], a @ wt.double(), (72 + 8) * U * (a.abs() @ wt.double().abs()))
    _within(got["bias"], a.sum(0), (M + 8) * U * a.abs().sum(0))
    assert not got["x"][:-tail].any()


def test_long_caches_of_keys():
    """Keys whose tokens lie 16 KB apart, 4.9 GB of them; the seen ones are the last."""
    need_gpu()
    r = _rnd(29)
    S, D, last = 300_000, 64, 200
    buf = torch.zeros(S, 2, 64, D, dtype=BF16, device="cuda")
    buf[-last:, :, 5] = r(last, 2, D).to(BF16)
    k, v = (buf[None, :, i, 5:6] for i in (0, 1))
    mask = torch.zeros(1, S, dtype=torch.bool, device="cuda")
    mask[:, -last:] = True
    for Sq in (1, 140):
        say("long cache", Sq)
        q, dout = r(1, Sq, 1, D).to(BF16), r(1, Sq, 1, D).to(BF16)
        lse = torch.empty(1, 1, Sq, device="cuda")
        out = kernels.cross_attention(q, k, v, key_mask=mask, lse=lse)
        short = [t[:, -last:] for t in (k, v)]
        seen = torch.ones(1, last, dtype=torch.bool, device="cuda")
        O, slack, _, grads = _cross_formula(q, *short, seen, D ** -0.5, dout)  # noqa: E741
        _within(out, O, slack)
        for name, g in zip(("dq", "dk", "dv"),
                           kernels.cross_attention_backward(dout, q, k, v, out, lse, key_mask=mask)):
            if name != "dq":
                assert not g[:, :-last].any()
                g = g[:, -last:]
            _within(g, grads[name][0], grads[name][1] + 1e-30)


# ---- cross attention -----------------------------------------------------------------------

CROSS = [
    # B, Sq, Sk, Hk, G, D, keys, type
    (1, 1, 1, 1, 1, 64, "all", BF16),
    (2, 1, 70, 2, 4, 128, "lens", FP16),
    (3, 33, 64, 5, 2, 64, "mask", BF16),
    (1, 128, 128, 2, 1, 128, "all", FP16),
    (3, 257, 77, 2, 3, 64, "lens", BF16),
    (2, 131, 513, 1, 1, 128, "mask", BF16),
    (4, 5, 1000, 1, 8, 128, "lens", BF16),       # keys in parts
    (1, 700, 3, 2, 1, 128, "all", BF16),
    (2, 3, 2500, 3, 1, 64, "mask", BF16),
    (5, 2, 66, 1, 7, 128, "both", BF16),
    (2, 4, 4000, 1, 8, 128, "mask", BF16),       # 32 rows: the last size of a wave a tile, in parts
    (1, 33, 1500, 1, 1, 64, "lens", BF16),       # the first over tiles of 128 rows
    (64, 1, 2100, 5, 1, 128, "mask", FP16),      # nine tiles a wave
    (130, 1, 300, 4, 2, 64, "both", BF16),       # two waves a workgroup
    (260, 2, 200, 2, 1, 128, "lens", FP16),
]


def _cross_case(B, Sq, Sk, Hk, G, D, keys, t, seed=0):
    r = _rnd(seed)
    q, k, v = r(B, Sq, Hk * G, D).to(t), r(B, Sk, Hk, D).to(t), r(B, Sk, Hk, D).to(t)
    kw = {}
    seen = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
    if keys in ("lens", "both"):
        lens = torch.tensor([max(0, Sk - b * (Sk + 2) // max(B - 1, 1)) for b in range(B)], dtype=torch.int32,
                            device="cuda")
        kw["kv_lens"] = lens
        seen = torch.arange(Sk, device="cuda") < lens[:, None]
    if keys in ("mask", "both"):
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        kw["key_mask"] = torch.rand(B, Sk, generator=g, device="cuda") < 0.6
        kw["key_mask"][-1] = False               # a stream that sees nothing
        seen = seen & kw["key_mask"]
    # what is not seen is not read
    k[~seen] = float("nan")
    v[~seen] = float("inf")
    return q, k, v, kw, seen, r(B, Sq, Hk * G, D).to(t)


def _cross_formula(q, k, v, seen, scale, dout):
    """64-bit results and the sums that their bounds are made of."""
    H, Hk, D = q.shape[2], k.shape[2], q.shape[3]
    heads = lambda t: t.double().transpose(1, 2)  # noqa: E731
    clean = lambda t: torch.where(seen[:, :, None, None], t.double(), torch.zeros((), device="cuda").double())  # noqa: E731
    Q, K, V, dO = heads(q), heads(clean(k)).repeat_interleave(H // Hk, 1), \
        heads(clean(v)).repeat_interleave(H // Hk, 1), heads(dout)
    S = (Q @ K.transpose(2, 3) * scale).masked_fill(~seen[:, None, None], float("-inf"))
    P = torch.nan_to_num(torch.softmax(S, -1))
    lse = torch.logsumexp(S, -1)
    step = _step(q.dtype)
    # scores in fp32: D products and the running maximum; a weight's relative error is theirs
    size = Q.abs() @ K.abs().transpose(2, 3) * scale
    dS_ = (D + 8) * U * 4 * (size + size.amax(-1, keepdim=True)) + 2.0 ** -20
    O = P @ V  # noqa: E741
    spread = (P * (step + dS_)) @ V.abs() + (P * (step + dS_)).sum(-1, keepdim=True) * O.abs()
    e_O = spread + (seen.shape[1] + 8) * U * (P @ V.abs())
    out_err = e_O + step * (O.abs() + e_O)
    # gradient: P from lse (its sum of rounded weights within a step), handed over and rounded
    e_P = P * (dS_ + step + (P * (step + dS_)).sum(-1, keepdim=True) + 2.0 ** -11) + 2.0 ** -24
    dP = dO @ V.transpose(2, 3)
    delta = (dO * O).sum(-1, keepdim=True)
    e_dP = (D + 8) * U * (dO.abs() @ V.abs().transpose(2, 3)) + \
        (dO.abs() * out_err).sum(-1, keepdim=True) + (D + 8) * U * (dO * O).abs().sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_dS = e_P * ((dP - delta).abs() + e_dP) + P * e_dP
    e_dS = e_dS + step * (dS.abs() + e_dS)
    e_dS, e_P = (torch.where(seen[:, None, None], t, torch.zeros_like(t)) for t in (e_dS, e_P))
    n = (q.shape[1] * (H // Hk) + 8) * U
    shared = lambda t: t.reshape(t.shape[0], Hk, H // Hk, *t.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
    grads = {
        "dq": ((dS @ K * scale).transpose(1, 2),
               ((e_dS + (seen.shape[1] + 8) * U * dS.abs()) @ K.abs() * scale).transpose(1, 2)),
        "dk": (shared(dS.transpose(2, 3) @ Q * scale),
               shared((e_dS + n * dS.abs()).transpose(2, 3) @ Q.abs() * scale)),
        "dv": (shared(P.transpose(2, 3) @ dO), shared((e_P + n * P).transpose(2, 3) @ dO.abs())),
    }
    return O.transpose(1, 2), e_O.transpose(1, 2), lse, grads


@pytest.mark.parametrize("B,Sq,Sk,Hk,G,D,keys,t", CROSS)
def test_cross_attention_matches_the_formula(B, Sq, Sk, Hk, G, D, keys, t):
    need_gpu()
    q, k, v, kw, seen, dout = _cross_case(B, Sq, Sk, Hk, G, D, keys, t)
    say("cross attention", B, Sq, Sk, Hk, G, D, keys, t)
    lse = torch.empty(B, Hk * G, Sq, device="cuda")
    got = kernels.cross_attention(q, k, v, lse=lse, **kw)
    O, slack, ref_lse, _ = _cross_formula(q, k, v, seen, 1 / math.sqrt(D), dout)  # noqa: E741
    _within(got, O, slack)
    none = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse), none) and bool((lse[none] < 0).all())
    assert not got.transpose(1, 2)[none].any()
    # the sum is of the rounded weights: within a step, and fp32 scores
    assert bool(((lse.double() - ref_lse)[~none].abs() <= 2 * _step(t) + 2.0 ** -18).all())


@pytest.mark.parametrize("B,Sq,Sk,Hk,G,D,keys,t", CROSS)
def test_cross_attention_gradients_match_the_formula(B, Sq, Sk, Hk, G, D, keys, t):
    need_gpu()
    if t == FP16:
        t = BF16
    q, k, v, kw, seen, dout = _cross_case(B, Sq, Sk, Hk, G, D, keys, t, seed=2)
    say("cross attention gradient", B, Sq, Sk, Hk, G, D, keys)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = kernels.cross_attention_train(*leaves, **kw)
    got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    again = torch.autograd.grad(out, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    _, _, _, grads = _cross_formula(q, k, v, seen, 1 / math.sqrt(D), dout)
    for name, g in zip(("dq", "dk", "dv"), got):
        ref, slack = grads[name]
        _within(g, ref, slack + 1e-30)
    for g in got[1:]:
        assert not g[~seen].any()


def test_cross_attention_gradient_matches_differences():
    need_gpu()
    q, k, v, kw, seen, dout = _cross_case(2, 24, 40, 2, 2, 64, "all", BF16, seed=5)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(kernels.cross_attention_train(*leaves), leaves, dout)
    r, h = _rnd(6), 1e-4
    along = [r(*x.shape).double() for x in leaves]

    def f(s):
        a = [x.double() + s * d for x, d in zip((q, k, v), along)]
        Q, K, V = a[0].transpose(1, 2), *(x.transpose(1, 2).repeat_interleave(2, 1) for x in a[1:])
        return (dout.double().transpose(1, 2) * (torch.softmax(Q @ K.transpose(2, 3) / 8, -1) @ V)).sum()
    want = float((f(h) - f(-h)) / (2 * h))
    have = float(sum((g.double() * d).sum() for g, d in zip(got, along)))
    size = math.sqrt(sum(float((g.double() * d).square().sum()) for g, d in zip(got, along)))
    assert abs(have - want) <= 6 * 4 * 2.0 ** -8 * size


def test_large_scores_keep_their_softmax():
    """Scores of 10^4 to 10^9, of either sign: one key takes all, ties are shared."""
    need_gpu()
    r = _rnd(21)
    for big in (1e4, 1e6, 1e9):
        for sign in (1, -1):
            q = torch.full((1, 40, 2, 64), 1.0, device="cuda", dtype=BF16)
            k = torch.zeros(1, 150, 2, 64, device="cuda", dtype=BF16)
            k[..., 0] = sign * big * (1 + torch.arange(150, device="cuda")[None, :, None] / 4).to(BF16)
            v = r(1, 150, 2, 64).to(BF16)
            s = k[0, :, 0, 0].double() / 8
            p = torch.softmax(s, 0)
            got = kernels.cross_attention(q, k, v)
            want = (p[:, None, None] * v[0].double()).sum(0)
            assert bool(((got[0].double() - want).abs() <= 2.0 ** -7 * (want.abs() + 1e-3)).all()), (big, sign)


def test_small_weights_count_in_the_sum():
    """One key whose score is far above thousands of equal others: their weights, subnormal in
    fp16, are in the sum as they are in the product."""
    need_gpu()
    S, D, R = 4096, 64, 66000            # rows enough that no split has a maximum of its own
    for t, gap in ((FP16, 11.0), (FP16, 14.0), (BF16, 14.0)):
        q, k = torch.zeros(1, R, 1, D, dtype=t, device="cuda"), torch.zeros(1, S, 1, D, dtype=t, device="cuda")
        q[..., 0], k[:, 1:, :, 0] = 8.0, -gap            # scores -gap at a scale of 1/8
        v = (1 + _rnd(5)(1, S, 1, D)).to(t)
        lse = torch.empty(1, 1, R, device="cuda")
        say("small weights", t, gap)
        out = kernels.cross_attention(q, k, v, lse=lse)
        w = torch.full((S,), -gap, dtype=torch.float64, device="cuda").exp()
        w[0] = 1.0
        want = (w[:, None] * v[0, :, 0].double()).sum(0) / w.sum()
        # weights: each off by half a step of the type, for fp16 below 2^-14 by at most 2^-25; both
        # enter O's numerator (|v| <= 6) and its sum, which is that of the rounded weights
        half = torch.finfo(t).eps / 2
        wobble = (half * w.sum() + S * (2.0 ** -25 if t == FP16 else 0.0)) / w.sum() * 2 * 6 + 2.0 ** -12
        err = (out[0, :, 0].double() - want).abs()
        assert bool((err <= half * want.abs() + wobble).all())
        assert bool((lse - w.sum().log()).abs().max() <= half + S * 2.0 ** -25 + 2.0 ** -12)


@pytest.mark.parametrize("Sq", [70, 4])
def test_growing_scores_refresh_the_maximum(Sq):
    """Every key block above the one before, the first keys masked."""
    need_gpu()
    r = _rnd(23)
    q = torch.ones(1, Sq, 1, 128, device="cuda", dtype=BF16)
    k = 0.05 * r(1, 640, 1, 128)
    k = (k + torch.arange(640, device="cuda")[None, :, None, None] / 80).to(BF16)
    v = r(1, 640, 1, 128).to(BF16)
    mask = torch.arange(640, device="cuda")[None] >= 96
    got = kernels.cross_attention(q, k, v, key_mask=mask)
    O, slack, _, _ = _cross_formula(q, k, v, mask, 1 / math.sqrt(128), torch.zeros_like(q))  # noqa: E741
    _within(got, O, slack)


@pytest.mark.parametrize("Sq", [1, 40, 200])
def test_keys_that_are_not_numbers_stay_in_their_stream(Sq):
    """A seen key or value that is NaN or infinite makes its stream's rows (that see it) so, no
    others, in one part or several; hidden ones nothing (the other tests' masked keys are NaN)."""
    need_gpu()
    r = _rnd(31)
    q, k, v = r(3, Sq, 2, 64).to(BF16), r(3, 3000, 2, 64).to(BF16), r(3, 3000, 2, 64).to(BF16)
    clean = kernels.cross_attention(q, k, v)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for which in (0, 1):
            kk, vv = k.clone(), v.clone()
            (kk, vv)[which][1, 2500, 1, 7] = bad
            say("not a number", Sq, bad, which)
            lse = torch.empty(3, 2, Sq, device="cuda")
            got = kernels.cross_attention(q, kk, vv, lse=lse)
            assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
            assert torch.equal(got[1, :, 0], clean[1, :, 0])
            P = torch.softmax((q[1, :, 1].float() @ kk[1, :, 1].float().t()) / 8, -1)
            want = P @ vv[1, :, 1].float()
            assert torch.equal(torch.isnan(got[1, :, 1]), torch.isnan(want))
            assert torch.equal(torch.isinf(got[1, :, 1]), torch.isinf(want))


def test_cross_attention_reads_views():
    """Heads of one projection, head-major storage, expanded streams and heads, odd addresses."""
    need_gpu()
    r = _rnd(25)
    qkv = r(2, 50, 3, 4, 64).to(BF16)
    q, k, v = qkv.unbind(2)
    want = kernels.cross_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(kernels.cross_attention(q, k, v), want)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(kernels.cross_attention(*major), want)
    odd = torch.zeros(2, 50, 4, 65, dtype=BF16, device="cuda")[..., 1:]
    odd.copy_(k)
    assert torch.equal(kernels.cross_attention(q, odd, v), want)
    one = kernels.cross_attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1))
    assert torch.equal(one, kernels.cross_attention(q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1)))
    same = kernels.cross_attention(q, k[:, :1].expand(-1, 50, -1, -1), v)
    assert torch.equal(same, kernels.cross_attention(q, k[:, :1].repeat(1, 50, 1, 1), v))
    # gradients of broadcast inputs are sums
    leaf = k[:1].clone().requires_grad_()
    dout = r(2, 50, 4, 64).to(BF16)
    got, = torch.autograd.grad(kernels.cross_attention_train(q, leaf.expand(2, -1, -1, -1), v), leaf, dout)
    full = k[:1].repeat(2, 1, 1, 1).requires_grad_()
    each, = torch.autograd.grad(kernels.cross_attention_train(q, full, v), full, dout)
    assert bool(((got.double() - each.double().sum(0, keepdim=True)).abs() <= 2.0 ** -8 * each.double().abs().sum(0)).all())
    # counts past the keys and below none
    lens = torch.tensor([99, -3], dtype=torch.int32, device="cuda")
    some = kernels.cross_attention(q, k, v, kv_lens=lens)
    assert torch.equal(some[:1], want[:1]) and not some[1].any()
    assert torch.equal(kernels.cross_attention(q, k, v, kv_lens=lens.long()), some)
    # nothing to see, nobody to look
    assert not kernels.cross_attention(q, k[:, :0], v[:, :0]).any()
    assert kernels.cross_attention(q[:, :0], k, v).shape == (2, 0, 4, 64)
    grads = kernels.cross_attention_backward(dout[:, :0], q[:, :0], k, v, q[:, :0],
                                             torch.empty(2, 4, 0, device="cuda"))
    assert not grads[1].any() and not grads[2].any()


# ---- streams, graphs ---------------------------------------------------------------------

def _block_step(x, ctx, p):
    """A run of the operators as a block uses them, without gradient."""
    y, h = kernels.rms_norm(x, p["g"], eps=1e-6, residual=p["r"])
    q = kernels.linear_act(y, p["wq"], p["b"]).unflatten(-1, (4, 64))
    k = kernels.linear_act(ctx, p["wk"], p["b"]).unflatten(-1, (4, 64))
    a = kernels.cross_attention(q, k, k, key_mask=p["mask"]).flatten(-2)
    return kernels.linear_act(a, p["wq"], p["b"], activation="gelu_tanh", residual=h, gate=p["gate"])


def _block_inputs(seed, S=200):
    r = _rnd(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = dict(g=1 + 0.1 * r(256), r=r(2, S, 256).to(BF16), wq=(r(256, 256) / 16).to(BF16), wk=(r(256, 256) / 16).to(BF16),
             b=r(256).to(BF16), gate=r(2, 2, 256).to(BF16), mask=torch.rand(2, 300, generator=g, device="cuda") < 0.7)
    return r(2, S, 256).to(BF16), r(2, 300, 256).to(BF16), p


def test_run_on_another_stream():
    need_gpu()
    x, ctx, p = _block_inputs(31)
    want = _block_step(x, ctx, p)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for s in (side, torch.cuda.current_stream()) * 3:
        with torch.cuda.stream(s):
            outs.append(_block_step(x, ctx, p))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("S", [2, 200])
def test_captured_run_replays(S):
    """Two graphs, replayed in turn with new inputs and eager work between."""
    need_gpu()
    sets = [_block_inputs(s, S) for s in (41, 42)]
    graphs = []
    for x, ctx, p in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _block_step(x, ctx, p)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block_step(x, ctx, p)
        graphs.append((graph, out))
    for i in range(4):
        for (x, ctx, p), (graph, out) in zip(sets, graphs):
            x.copy_(_rnd(50 + i)(*x.shape).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, _block_step(x, ctx, p)), i


def test_captured_training_step_replays():
    need_gpu()
    x, ctx, p = _block_inputs(61)
    w = p["wq"].clone().requires_grad_()
    dy = _rnd(62)(2, 200, 256).to(BF16)

    def step():
        y, h = kernels.rms_norm_train(x, p["g"], eps=1e-6, residual=p["r"])
        q = kernels.linear_act_train(y, w, p["b"]).unflatten(-1, (4, 64))
        k = kernels.linear_act_train(ctx, w, p["b"]).unflatten(-1, (4, 64))
        a = kernels.cross_attention_train(q, k, k, key_mask=p["mask"]).flatten(-2)
        out = kernels.linear_act_train(a, w, p["b"], activation="gelu_tanh", residual=h, gate=p["gate"])
        return torch.autograd.grad(out, w, dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(_rnd(70 + i)(*x.shape).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step()), i


# ---- modules -------------------------------------------------------------------------------

def test_block_modules_against_torch_in_64_bits():
    """Cross attention, norm and feed-forward as a block runs them: values and every
    parameter's gradient; the bf16 run against the same modules in 64 bits."""
    need_gpu()
    torch.manual_seed(3)
    dim, heads, S, Sc = 256, 4, 90, 33
    attn, ffn = CrossAttention(dim, heads).cuda(), FeedForward(dim, 512).cuda()
    for m in (attn, ffn):
        m.to(BF16)
    wide_attn, wide_ffn = CrossAttention(dim, heads).cuda().double(), FeedForward(dim, 512).cuda().double()
    for a, b in ((attn, wide_attn), (ffn, wide_ffn)):
        b.load_state_dict({k: v.double() for k, v in a.state_dict().items()})
    wide_attn.norm_q, wide_attn.norm_k = (_WideNorm(n) for n in (wide_attn.norm_q, wide_attn.norm_k))
    r = _rnd(4)
    x, ctx, gate = r(2, S, dim).to(BF16), r(2, Sc, dim).to(BF16), r(2, 3, dim).to(BF16)
    lens = torch.tensor([33, 12], dtype=torch.int32, device="cuda")
    dy = r(2, S, dim).to(BF16)

    def run(attn, ffn, t):
        X = x.to(t).requires_grad_()
        h = attn(X, ctx.to(t), kv_lens=lens, residual=X)
        y = ffn(h, residual=h, gate=gate.to(t))
        params = [X, *attn.parameters(), *ffn.parameters()]
        return y, torch.autograd.grad(y, params, dy.to(t))
    y, grads = run(attn, ffn, BF16)
    kept = []
    wide_attn.k.register_forward_hook(lambda m, i, o: kept.append(o))
    wide, wide_grads = run(wide_attn, wide_ffn, torch.float64)
    # a dozen roundings in a row, each 2^-8 of its values, and products that average them:
    # 2^-5 in the norm bounds their sum.  For k's bias that is relative to the rows' terms, not to
    # their sum: a row of dS adds up to 0, so sum_k dS q = 0 for every q, and what is left of the
    # keys' sum is only how the norm's factor differs from key to key
    name_of = ["x"] + [f"attn.{n}" for n, _ in attn.named_parameters()] + [f"ffn.{n}" for n, _ in ffn.named_parameters()]
    h = wide_attn(x.double(), ctx.double(), kv_lens=lens, residual=x.double())
    dk, = torch.autograd.grad(wide_ffn(h, residual=h, gate=gate.double()), kept.pop(), dy.double())
    for name, a, b in (("y", y, wide), *zip(name_of, grads, wide_grads)):
        size = dk.abs().sum((0, 1)) if name == "attn.k.bias" else b
        assert float((a.double() - b).detach().norm()) <= 2.0 ** -5 * float(size.detach().norm()) + 1e-6, name
    with torch.no_grad():
        kv = attn.project_context(ctx)
        again = ffn(attn(x, kv=kv, kv_lens=lens, residual=x), residual=attn(x, ctx, kv_lens=lens, residual=x), gate=gate)
        assert torch.equal(again, y.detach())


class _WideNorm(RMSNorm):
    def __init__(self, norm):
        super().__init__(norm.weight.numel(), norm.eps)
        self.weight = norm.weight

    def forward(self, x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight


# ---- refusals ------------------------------------------------------------------------------

def test_refusals():
    need_gpu()
    r = _rnd(90)
    x, w = r(4, 64).to(BF16), r(32, 64).to(BF16)
    bad = [
        (ValueError, lambda: kernels.linear_act(x, w[:, :32])),
        (ValueError, lambda: kernels.linear_act(x, w.half())),
        (ValueError, lambda: kernels.linear_act(x, w, r(31).to(BF16))),
        (ValueError, lambda: kernels.linear_act(x, w, activation="relu6")),
        (ValueError, lambda: kernels.linear_act(x, w, gate=r(3, 32).to(BF16))),
        (ValueError, lambda: kernels.linear_act(x, w, residual=x)),
        (ValueError, lambda: kernels.linear_act(x, w, out=torch.empty(8, 32, dtype=BF16, device="cuda")[::2])),
        (ValueError, lambda: kernels.linear_act(x, w.cpu())),
        (ValueError, lambda: kernels.linear_act(x, r(64, 64).to(BF16), out=x)),
        (ValueError, lambda: kernels.linear_act(x[1:], r(64, 64).to(BF16), out=x[:3])),
        (ValueError, lambda: kernels.linear_act_backward(r(4, 32).to(BF16), x, w, activation="silu")),
        (NotImplementedError, lambda: kernels.linear_act(x.float(), w.float())),
        (RuntimeError, lambda: kernels.linear_act(x, w.clone().requires_grad_())),
        (ValueError, lambda: kernels.rms_norm(x, r(63), eps=1e-6)),
        (ValueError, lambda: kernels.rms_norm(x, r(64), eps=-1.0)),
        (ValueError, lambda: kernels.rms_norm(x, r(64), eps=float("nan"))),
        (ValueError, lambda: kernels.rms_norm(x, r(64), eps=1e-6, residual=x[:2])),
        (NotImplementedError, lambda: kernels.rms_norm(r(2, 16392).to(BF16), r(16392), eps=1e-6)),
        (NotImplementedError, lambda: kernels.rms_norm(x.float(), r(64), eps=1e-6)),
    ]
    q, k = r(2, 5, 4, 64).to(BF16), r(2, 9, 2, 64).to(BF16)
    lens, mask = torch.tensor([9, 9], dtype=torch.int32, device="cuda"), torch.ones(2, 9, dtype=torch.bool, device="cuda")
    bad += [
        (ValueError, lambda: kernels.cross_attention(q, k, k[:, :8])),
        (ValueError, lambda: kernels.cross_attention(q[:, :, :3], k, k)),
        (ValueError, lambda: kernels.cross_attention(q[0], k, k)),
        (ValueError, lambda: kernels.cross_attention(q, k.half(), k)),
        (NotImplementedError, lambda: kernels.cross_attention(q[..., :32], k[..., :32], k[..., :32])),
        (ValueError, lambda: kernels.cross_attention(q, k, k, kv_lens=lens[:1])),
        (ValueError, lambda: kernels.cross_attention(q, k, k, kv_lens=lens.cpu())),
        (ValueError, lambda: kernels.cross_attention(q, k, k, kv_lens=lens.float())),
        (ValueError, lambda: kernels.cross_attention(q, k, k, key_mask=mask[:, :8])),
        (ValueError, lambda: kernels.cross_attention(q, k, k, key_mask=mask.int())),
        (ValueError, lambda: kernels.cross_attention(q, k, k, scale=-1.0)),
        (ValueError, lambda: kernels.cross_attention(q, k, k, scale=float("nan"))),
        (ValueError, lambda: kernels.cross_attention(q, k, k, out=q[:1].expand(2, -1, -1, -1))),
        (ValueError, lambda: kernels.cross_attention(q, k, k, out=q)),
        (ValueError, lambda: kernels.cross_attention(k, k, k, out=k)),
        (ValueError, lambda: kernels.cross_attention(q, k, k, lse=torch.empty(2, 4, 6, device="cuda"))),
        (RuntimeError, lambda: kernels.cross_attention(q.clone().requires_grad_(), k, k)),
        (NotImplementedError, lambda: kernels.cross_attention_train(q.half().requires_grad_(), k.half(), k.half())),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")
