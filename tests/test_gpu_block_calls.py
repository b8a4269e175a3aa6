"""Calls of the block's operators that their documentation allows and the formulas' cases
do not make, against the formulas in 64 bits.  Bounds as in ``test_gpu_block``."""

import copy
import math

import pytest
import torch

from multics_amd import _capi, block, kernels
from multics_amd.module import CrossAttention, FeedForward, _gated
from tests.gpu_util import need_gpu, say
from tests.test_block import CHANGES, EPILOGUES, _Adapter, change_ffn
from tests.test_gpu_block import BF16, FP16, U, _act64, _linear_case, _rnd, _step, _within

pytestmark = pytest.mark.gpu


# ---- values that are not numbers --------------------------------------------------------

@pytest.mark.parametrize("t,N", [(BF16, 264), (FP16, 264), (BF16, 77)])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
def test_gradient_of_a_nan_before_the_activation(act, t, N):
    """It reaches the gradients of its row and its channel, and no others."""
    need_gpu()
    M, K = 150, 64
    x, w, b, _, gate, dy = _linear_case(M, K, N, act, 3, False, t)
    z = (x.float() @ w.float().t() + b.float()).to(t)
    say("a NaN before the activation", act, t, N)
    clean = kernels.linear_act_backward(dy, x, w, preact=z, activation=act, gate=gate)
    z[70, 5] = float("nan")
    got = kernels.linear_act_backward(dy, x, w, preact=z, activation=act, gate=gate)
    rows = torch.arange(M, device="cuda") != 70
    cols = torch.arange(N, device="cuda") != 5
    assert torch.isnan(got["x"][70]).all() and torch.equal(got["x"][rows], clean["x"][rows])
    assert torch.isnan(got["weight"][5]).all() and torch.equal(got["weight"][cols], clean["weight"][cols])
    assert torch.isnan(got["bias"][5]) and torch.equal(got["bias"][cols], clean["bias"][cols])
    assert torch.isnan(got["gate"][1, 5])                    # (50 rows a gate)
    got["gate"][1, 5] = clean["gate"][1, 5]
    assert torch.equal(got["gate"], clean["gate"])


@pytest.mark.parametrize("M,N", [(6, 40), (33, 40), (140, 264), (140, 77)])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
def test_gate_gradient_of_values_below_fp16(act, M, N):
    """Far below what fp16 holds every activation is 0: the gate's gradient is that of
    the other rows, not a NaN of -inf * 0."""
    need_gpu()
    r = _rnd(7)
    x, w = torch.zeros(M, 8, dtype=FP16, device="cuda"), torch.zeros(N, 8, dtype=FP16, device="cuda")
    x[:, 0], w[:, 0] = r(M).to(FP16), r(N).to(FP16)
    x[2, 1], w[::3, 1] = 1000.0, -100.0                      # row 2: z about -10^5 in every third channel
    gate, dy = r(N).to(FP16).requires_grad_(), r(M, N).to(FP16)
    say("values below fp16", act, M, N)
    y = kernels.linear_act_train(x, w, activation=act, gate=gate)
    got, = torch.autograd.grad(y, gate, dy)
    z = x.double() @ w.double().t()
    a, size = _act64(z, act), z.abs() * (z > -1e4)           # (exactly 0 below)
    step = _step(FP16)
    # z as kept: one rounding; the sum over M rows
    terms = dy.double().abs() * (1.2 * step * size + 2.0 ** -25 + 2.0 ** -19 * size + (M + 16) * U * a.abs())
    _within(got, (dy.double() * a).sum(0), terms.sum(0))


# ---- rows far apart ---------------------------------------------------------------------

@pytest.mark.parametrize("B,S,K,N,act", [(4, 4620, 1536, 200, "gelu_tanh"), (70, 1400, 1536, 136, "silu"),
                                         (3, 2100, 1001, 33, None)])
def test_product_of_rows_far_apart(B, S, K, N, act):
    """The last token of every stream: rows two million elements apart and more."""
    need_gpu()
    r = _rnd(15)
    buf = torch.zeros(B, S, K, dtype=BF16, device="cuda")
    buf[:, -1] = r(B, K).to(BF16)
    x = buf[:, -1]
    assert x.stride(0) >= 1 << 21
    w, b, dy = (r(N, K) / math.sqrt(K)).to(BF16), r(N).to(BF16), r(B, N).to(BF16)
    far = torch.zeros(N, 1 << 21, dtype=BF16, device="cuda")[:, :K] if N == 33 else w    # weights too
    far.copy_(w)
    say("rows far apart", B, S, K, N, act)
    assert torch.equal(kernels.linear_act(x, far, b, activation=act),
                       kernels.linear_act(x.contiguous(), w, b, activation=act))
    grads = []
    for rows, weights in ((x, far), (x.contiguous(), w)):
        leaves = [t.detach().requires_grad_() for t in (rows, weights, b)]
        grads.append(torch.autograd.grad(kernels.linear_act_train(*leaves, activation=act), leaves, dy))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_weights_gradient_of_one_row_at_a_stride_of_0():
    """The C entry: an infinity of the only row is one in dw (the rows past it are not that row)."""
    need_gpu()
    x, w = torch.zeros(1, 64, dtype=BF16, device="cuda"), torch.ones(32, 64, dtype=BF16, device="cuda")
    x[0, 3], x[0, 4] = float("inf"), 2.0
    dy, dw = torch.ones(1, 32, dtype=BF16, device="cuda"), torch.empty(32, 64, dtype=BF16, device="cuda")
    fields = (1, 32, 64, 0, 0, x.data_ptr(), w.data_ptr(), 0, dy.data_ptr(), 0, 0, dw.data_ptr(), 0, 0, 0, 64, 0, 32, 0,
              64, 64, 1)
    size = block._workspace("hier_linear_bwd_workspace", block._pack_linear_bwd(*fields, 0, 0))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    _capi.call_on(x.device, "hier_linear_bwd", block._pack_linear_bwd(*fields, ws.data_ptr(), size))
    assert torch.equal(dw, x.expand(32, 64))


# ---- what a gradient reads ----------------------------------------------------------------

@pytest.mark.parametrize("need,rows", [(("bias", "gate"), None), (("x",), (0, 33)), (("weight",), (50, 0)),
                                       (("x", "weight"), (50, 33))])
def test_gradient_copies_what_it_reads(need, rows, monkeypatch):
    """Odd channels: x is copied to whole rows for the weights' gradient alone, the weights for x's."""
    need_gpu()
    x, w, b, _, gate, dy = _linear_case(50, 77, 33, None, 2, False, BF16)
    z = (x.float() @ w.float().t()).to(BF16)
    want = kernels.linear_act_backward(dy, x, w, preact=z, gate=gate)
    seen = []
    pack = block._pack_pad

    def spy(*fields):
        seen.append(fields[:2])
        return pack(*fields)
    monkeypatch.setattr(block, "_pack_pad", spy)
    got = kernels.linear_act_backward(dy, x, w, preact=z, gate=gate, need=need)
    assert set(got) == set(need) and all(torch.equal(got[n], want[n]) for n in need)
    assert seen == ([] if rows is None else [rows])


# ---- small weights of the attention's gradient ----------------------------------------------

@pytest.mark.parametrize("Sq,Sk,peak,D", [(40, 4096, 14.0, 64), (40, 4096, 20.0, 128), (2000, 300, 18.0, 128),
                                          (200, 65536, None, 64)])
def test_gradient_of_keys_of_small_weight(Sq, Sk, peak, D):
    """Thousands of keys beside one that takes most of the weight, or of even weight: their
    gradients to the precision of bf16, however small the weights."""
    need_gpu()
    r = _rnd(19)
    scale = D ** -0.5
    q, k = r(1, Sq, 1, D), 0.25 * r(1, Sk, 1, D)
    if peak is not None:
        q[..., 0], k[..., 0] = 4.0, 0.0
        k[:, 3] = 0.0
        k[:, 3, :, 0] = peak / (4.0 * scale)
    q, k, v, dout = q.to(BF16), k.to(BF16), r(1, Sk, 1, D).to(BF16), r(1, Sq, 1, D).to(BF16)
    say("keys of small weight", Sq, Sk, peak, D)
    lse = torch.empty(1, 1, Sq, device="cuda")
    out = kernels.cross_attention(q, k, v, lse=lse)
    dq, dk, dv = kernels.cross_attention_backward(dout, q, k, v, out, lse)
    Q, K, V, dO = (t[0, :, 0].double() for t in (q, k, v, dout))
    S = Q @ K.t() * scale
    P = torch.softmax(S, -1)
    step = _step(BF16)
    size = Q.abs() @ K.abs().t() * scale
    e_S = (D + 8) * U * 4 * (size + size.amax(-1, keepdim=True)) + 2.0 ** -20
    O = P @ V  # noqa: E741
    e_O = (P * (step + e_S)) @ V.abs() + (P * (step + e_S)).sum(-1, keepdim=True) * O.abs() + (Sk + 8) * U * (P @ V.abs())
    e_O = e_O + step * (O.abs() + e_O)
    # P: of scores in fp32 and a sum of rounded weights; handed over in eleven bits, down to 2^-29
    e_P = P * (e_S + step + (P * (step + e_S)).sum(-1, keepdim=True) + 2.0 ** -11) + 2.0 ** -40
    dP, delta = dO @ V.t(), (dO * O).sum(-1, keepdim=True)
    e_dP = (D + 8) * U * (dO.abs() @ V.abs().t() + (dO * O).abs().sum(-1, keepdim=True)) + \
        (dO.abs() * e_O).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_dS = e_P * ((dP - delta).abs() + e_dP) + P * e_dP
    e_dS = e_dS + step * (dS.abs() + e_dS)
    n = (Sq + 8) * U
    _within(dk[0, :, 0], dS.t() @ Q * scale, (e_dS + n * dS.abs()).t() @ Q.abs() * scale + 1e-30)
    _within(dv[0, :, 0], P.t() @ dO, (e_P + n * P).t() @ dO.abs() + 1e-30)
    _within(dq[0, :, 0], dS @ K * scale, (e_dS + (Sk + 8) * U * dS.abs()) @ K.abs() * scale + 1e-30)
    if peak is not None:                       # and no key's gradient is lost
        ref = dS.t() @ Q * scale
        err = (dk[0, :, 0].double() - ref).norm(dim=-1) / ref.norm(dim=-1)
        err[3] = 0.0
        # three roundings (O, dS, the result) of at most a step of the terms, at random over rows and
        # channels: the terms' root of squares is within 1.5 of the sum's norm
        assert float(err.max()) <= 1.5 * math.sqrt(3) * step, float(err.max())


# ---- outputs that are given --------------------------------------------------------------

def test_outputs_in_the_memory_of_inputs():
    """Refused wherever a row that is written may be read; slices of one projection pass."""
    need_gpu()
    r = _rnd(29)
    x, w, buf = r(40, 64).to(BF16), r(72, 64).to(BF16), r(41, 72).to(BF16)
    square = r(64, 64).to(BF16)
    wide = r(40, 128).to(BF16)
    for call in (lambda: kernels.linear_act(x, w, residual=buf[1:], out=buf[:-1]),
                 lambda: kernels.linear_act(x, w, residual=buf[:1].expand(40, 72), out=buf[:-1]),
                 lambda: kernels.linear_act(x, w, gate=buf[0], out=buf[:-1]),
                 lambda: kernels.linear_act(x, w, buf[7], out=buf[:-1]),
                 lambda: kernels.linear_act(wide[:, :64], square, out=wide.view(80, 64)[:40])):
        with pytest.raises(ValueError, match="share memory"):
            call()
    qkv = r(2, 50, 3, 4, 64).to(BF16)
    q, k, v = qkv.unbind(2)
    lse = torch.empty(2, 4, 50, device="cuda")
    floats = torch.empty(2 * 50 * 4 * 32, device="cuda")
    cases = [dict(out=q), dict(out=k), dict(out=v),
             dict(out=q.flip(1).contiguous(), lse=qkv.view(-1).view(torch.float32)[:400].view(2, 4, 50)),
             dict(out=floats.view(BF16).view(2, 50, 4, 64), lse=floats[:400].view(2, 4, 50))]
    for kw in cases:
        with pytest.raises(ValueError, match="share memory"):
            kernels.cross_attention(q, k, v, **kw)
    # a fourth slice beside the three
    want = kernels.cross_attention(q, k, v)
    four = torch.zeros(2, 50, 4, 4, 64, dtype=BF16, device="cuda")
    four[:, :, :3] = qkv
    q, k, v, out = four.unbind(2)
    assert kernels.cross_attention(q, k, v, out=out, lse=lse) is out
    assert torch.equal(out, want) and torch.equal(four[:, :, :3], qkv)
    # the residual itself, also as rows of a larger tensor
    res = buf[3:].clone()
    got = kernels.linear_act(x[:38], w, residual=buf[3:], out=buf[3:])
    assert torch.equal(got, kernels.linear_act(x[:38], w, residual=res))


# ---- modules -------------------------------------------------------------------------------

@pytest.mark.parametrize("how", CHANGES)
def test_feed_forward_with_changed_children(how):
    need_gpu()
    torch.manual_seed(1)
    ffn = FeedForward(64, 128)
    change_ffn(ffn, how)
    ffn = ffn.cuda().to(BF16)
    x, res = _rnd(1)(3, 20, 64).to(BF16), _rnd(2)(3, 20, 64).to(BF16)
    y = ffn(x, residual=res)
    want = res + torch.nn.Sequential.forward(ffn, x)
    with torch.no_grad():
        assert torch.equal(ffn(x, residual=res), y)
    if how == "none":           # y rounds h and itself, the other h (twice), z and itself: three steps of it
        size = want.double().abs() + res.double().abs() + 8
        assert bool(((y.double() - want.double()).abs() <= 4 * 2.0 ** -8 * size).all())
    else:
        assert torch.equal(y, want)


@pytest.mark.parametrize("how", ["o adapter", "o hook", "q adapter", "norm", "norm hook", "none"])
def test_cross_attention_with_changed_children(how):
    """Against the same module on the host in fp32."""
    need_gpu()
    torch.manual_seed(2)
    host = CrossAttention(128, 2)
    if how in ("o adapter", "q adapter"):
        child = _Adapter(getattr(host, how[0]))
        if how == "q adapter":
            type(child).weight, kept = property(lambda self: 1 / 0), type(child).weight      # nobody looks at it
        setattr(host, how[0], child)
    elif how == "o hook":
        host.o.register_forward_hook(lambda m, i, o: 2 * o)
    elif how == "norm":
        host.norm_q = torch.nn.LayerNorm(128)
    elif how == "norm hook":
        host.norm_k.register_forward_hook(lambda m, i, o: 3 * o)
    try:
        gpu = copy.deepcopy(host).cuda().to(BF16)
        host.load_state_dict({k: v.float().cpu() for k, v in gpu.state_dict().items()})
        x, ctx, gate = _rnd(1)(2, 20, 128).to(BF16), _rnd(2)(2, 9, 128).to(BF16), _rnd(3)(2, 4, 128).to(BF16)
        with torch.no_grad():
            for kw in (dict(), dict(residual=x, gate=gate)):
                want = host(x.float().cpu(), ctx.float().cpu(), **{k: v.float().cpu() for k, v in kw.items()})
                y = gpu(x, ctx, **kw)
                # some ten roundings in a row of 2^-8 each, in the norm (a dropped child moves it by half)
                assert float((y.double().cpu() - want).norm()) <= 10 * 2.0 ** -8 * float(want.norm())
    finally:
        if how == "q adapter":
            type(child).weight = kept


@pytest.mark.parametrize("residual,gate,fits", EPILOGUES)
def test_modules_with_residuals_and_gates_of_other_types_and_shapes(residual, gate, fits):
    """An fp32 residual stream or gate, broadcast ones: as on the host, in the wider type."""
    need_gpu()
    torch.manual_seed(3)
    ffn, attn = FeedForward(8, 32).cuda().to(BF16), CrossAttention(128, 2).cuda().to(BF16)
    r = _rnd(4)
    for module, dim in ((ffn, 8), (attn, 128)):
        make = lambda what: None if what is None else r(*(dim if n == 8 else n for n in what[0])).to(  # noqa: E731, B023
            torch.float32 if what[1] == "wide" else BF16)
        res, g = make(residual), make(gate)
        args = (r(2, 6, dim).to(BF16),) + ((r(2, 5, dim).to(BF16),) if module is attn else ())
        say("residual and gate", residual, gate, dim)
        y = module(*args, residual=res, gate=g)
        want = _gated(module(*args), res, g)
        assert y.dtype == want.dtype and y.shape == want.shape
        # the bare product rounds to bf16 before the gate, the epilogue after it, and the sum
        # again: a step of the product at most, and one of the sum
        slack = (want.double() - (0 if res is None else res.double())).abs() + want.double().abs()
        assert bool(((y.double() - want.double()).abs() <= 2.0 ** -7 * slack + 1e-6).all())


@pytest.mark.parametrize("how", ["autocast", "fp16"])
def test_cross_attention_of_wider_weights_and_of_fp16_trains(how):
    """fp32 weights under autocast (the projections' bf16 goes to the kernels), and fp16 with
    gradients (torch operations), NaN in hidden states: against the module in 64 bits."""
    need_gpu()
    torch.manual_seed(5)
    attn = CrossAttention(128, 2).cuda()
    if how == "fp16":
        attn = attn.half()
    wide = copy.deepcopy(attn).double()
    t = torch.float32 if how == "autocast" else FP16
    x, ctx, dy = _rnd(1)(2, 20, 128).to(t), _rnd(2)(2, 9, 128).to(t), _rnd(3)(2, 20, 128).to(t)
    lens = torch.tensor([9, 4], device="cuda", dtype=torch.int32)

    def run(attn, x, ctx, dy, cast, bad):
        x = x.clone().requires_grad_()
        with torch.autocast("cuda", torch.bfloat16, enabled=cast):
            k, v = attn.project_context(ctx)
            hide = torch.arange(9, device="cuda")[None, :, None, None] >= lens[:, None, None, None]
            k, v = (torch.where(hide, torch.full_like(u, bad), u) for u in (k, v))
            y = attn(x, kv=(k, v), kv_lens=lens, residual=x)
        return y, torch.autograd.grad(y, [x, *attn.parameters()], dy.to(y.dtype))
    y, grads = run(attn, x, ctx, dy, how == "autocast", float("nan"))
    ref, want = run(wide, x.double(), ctx.double(), dy.double(), False, 0.0)
    # some ten roundings in a row, in the norm; the module's own norm is fp32 inside, hence 2^-18
    step = _step(BF16 if how == "autocast" else FP16)
    names = ["x", *(n for n, _ in attn.named_parameters())]
    assert float((y.detach().double() - ref).detach().norm()) <= 10 * step * float(ref.detach().norm())
    for name, a, b in zip(names, grads, want):
        if name != "k.bias":            # (zero but for the norm's change from key to key)
            assert float((a.double() - b).norm()) <= (16 * step + 2.0 ** -18) * float(b.norm()), name


# ---- many rows ---------------------------------------------------------------------------

def test_norm_of_more_rows_than_a_line_of_threads():
    """2^26 rows and a few: 2^32 threads, more than a launch takes side by side."""
    need_gpu()
    few, M = 1 << 16, (1 << 26) + 37
    r = _rnd(33)
    base, w = r(few, 8).to(BF16), 1 + 0.1 * r(8)
    x = base.repeat(M // few + 1, 1)[:M]
    say("norm of many rows", M)
    want = kernels.rms_norm(base, w, eps=1e-6)
    got = kernels.rms_norm(x, w, eps=1e-6)
    assert torch.equal(got[:-37].view(-1, few, 8), want.expand(M // few, few, 8))
    assert torch.equal(got[-37:], want[:37])
