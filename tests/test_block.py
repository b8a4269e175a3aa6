"""The block's operators without a GPU: what their C entries and Python calls refuse, and the
modules' torch path."""

import ctypes as C
import math

import pytest
import torch

from multics_amd import _capi, block, kernels, module
from multics_amd.module import CompatibleLinear, CrossAttention, FeedForward, RMSNorm

AT = 1 << 20             # an aligned address that nothing reads: the calls refuse before a launch


def _norm(**kw):
    f = dict(M=4, C=64, eps=1e-6, type=0, gain_type=2, x=AT, w=AT, y=AT, x_ss=64, y_ss=64)
    return _capi.HierRmsNormArgs(**{**f, **kw})


def _linear(**kw):
    f = dict(M=100, N=48, K=64, type=0, act=0, x=AT, w=AT, out=AT, x_ss=64, w_ss=64, out_ss=48, rows_per_gate=1)
    return _capi.HierLinearArgs(**{**f, **kw})


def _linear_bwd(**kw):
    f = dict(M=100, N=48, K=64, type=0, act=0, x=AT, w=AT, dy=AT, dx=AT, dw=AT, x_ss=64, w_ss=64, dy_ss=48,
             dx_ss=64, dw_ss=64, rows_per_gate=1)
    return _capi.HierLinearBwdArgs(**{**f, **kw})


def _cross(**kw):
    f = dict(B=2, Hq=4, Hk=2, D=64, type=0, scale=0.125, Sq=1000, Sk=9, q=AT, k=AT, v=AT, o=AT, lse=AT,
             q_sb=256000, q_ss=256, q_sh=64, k_sb=1152, k_ss=128, k_sh=64, v_sb=1152, v_ss=128, v_sh=64,
             o_sb=256000, o_ss=256, o_sh=64)
    return _capi.HierCrossArgs(**{**f, **kw})


def _pad(**kw):
    f = dict(rows0=3, rows1=2, ss0=7, ss1=7, src0=AT, src1=AT, dst0=AT, dst1=AT, C=7)
    return _capi.HierPadRowsArgs(**{**f, **kw})


@pytest.fixture(autouse=True)
def _no_error_left():
    """Whatever test runs next in this process finds no refusal of these."""
    yield
    args = _linear(M=0)
    assert _capi.lib().hier_linear(C.addressof(args), None) == 0


REFUSED = [
    ("hier_rms_norm", _norm, dict(C=0), "invalid"),
    ("hier_rms_norm", _norm, dict(C=16385, x_ss=16385, y_ss=16385), "16384"),
    ("hier_rms_norm", _norm, dict(type=2), "bf16 or fp16"),
    ("hier_rms_norm", _norm, dict(gain_type=7), "gain"),
    ("hier_rms_norm", _norm, dict(eps=float("nan")), "eps"),
    ("hier_rms_norm", _norm, dict(eps=-1.0), "eps"),
    ("hier_rms_norm", _norm, dict(x=None), "NULL"),
    ("hier_rms_norm", _norm, dict(r=AT), "NULL"),
    ("hier_rms_norm", _norm, dict(y_ss=8), "stride"),
    ("hier_linear", _linear, dict(K=60), "multiple of 8"),
    ("hier_linear", _linear, dict(N=0), "invalid"),
    ("hier_linear", _linear, dict(act=9), "activation"),
    ("hier_linear", _linear, dict(type=2), "bf16 or fp16"),
    ("hier_linear", _linear, dict(x=AT + 2), "aligned"),
    ("hier_linear", _linear, dict(w_ss=60), "stride"),
    ("hier_linear", _linear, dict(x_ss=1 << 21), "stride"),
    ("hier_linear", _linear, dict(out=None), "NULL"),
    ("hier_linear", _linear, dict(out_ss=40), "stride"),
    ("hier_linear", _linear, dict(gate=AT, rows_per_gate=0), "rows_per_gate"),
    ("hier_linear", _linear, dict(M=200, N=64, K=1 << 16, x_ss=1 << 16, w_ss=1 << 16, out_ss=64), "workspace"),
    ("hier_linear_bwd", _linear_bwd, dict(act=1), "before the activation"),
    ("hier_linear_bwd", _linear_bwd, dict(N=44, dy_ss=45), "workspace"),     # dy's rows are copied
    ("hier_pad_rows", _pad, dict(C=0), "invalid"),
    ("hier_pad_rows", _pad, dict(rows0=-1), "invalid"),
    ("hier_pad_rows", _pad, dict(dst0=AT + 2), "aligned"),
    ("hier_pad_rows", _pad, dict(src0=None), "rows"),
    ("hier_pad_rows", _pad, dict(ss1=-3), "strides"),
    ("hier_linear_bwd", _linear_bwd, dict(dgate=AT), "without a gate"),
    ("hier_linear_bwd", _linear_bwd, dict(gate=AT, rows_per_gate=33, preact=AT, preact_ss=48), "rows_per_gate"),
    ("hier_linear_bwd", _linear_bwd, dict(dy=None), "dy"),
    ("hier_linear_bwd", _linear_bwd, dict(dx_ss=8), "stride"),
    ("hier_linear_bwd", _linear_bwd, dict(db=AT), "workspace"),
    ("hier_linear_bwd", _linear_bwd, dict(x_ss=0, db=AT), "overlap"),
    ("hier_linear_bwd", _linear_bwd, dict(w_ss=0, db=AT), "overlap"),
    ("hier_linear_bwd", _linear_bwd, dict(w_ss=0, dx=None, db=AT), "workspace"),
    ("hier_linear_bwd", _linear_bwd, dict(x_ss=0, M=1, db=AT), "workspace"),
    ("hier_cross_attn", _cross, dict(D=32), "head_dim"),
    ("hier_cross_attn", _cross, dict(Hq=5), "invalid"),
    ("hier_cross_attn", _cross, dict(type=2), "bf16 or fp16"),
    ("hier_cross_attn", _cross, dict(scale=0.0), "scale"),
    ("hier_cross_attn", _cross, dict(scale=float("nan")), "scale"),
    ("hier_cross_attn", _cross, dict(q=AT + 8), "aligned"),
    ("hier_cross_attn", _cross, dict(k_ss=60), "16-byte rows"),
    ("hier_cross_attn", _cross, dict(k_ss=32), "overlap"),
    ("hier_cross_attn", _cross, dict(k_ss=1 << 23), "stride"),
    ("hier_cross_attn", _cross, dict(o_ss=0), "rows of its own"),
    ("hier_cross_attn", _cross, dict(v=None), "NULL"),
    ("hier_cross_attn", _cross, dict(Sq=1, Sk=8192), "workspace"),
    ("hier_cross_attn", _cross, dict(Sq=1 << 30), "too many"),
]


@pytest.mark.parametrize("name,make,change,says", REFUSED)
def test_entries_refuse(name, make, change, says):
    args = make(**change)
    rc = getattr(_capi.lib(), name)(C.addressof(args), None)
    assert rc < 0
    assert says in _capi.lib().hier_last_error().decode()


@pytest.mark.parametrize("change,says", [
    (dict(type=1), "bf16 only"), (dict(lse=None), "NULL"), (dict(q_sh=1 << 29), "too large"),
    (dict(), "workspace")])
def test_cross_gradient_entry_refuses(change, says):
    args = _capi.HierCrossBwdArgs(f=_cross(**change), dout=AT, dq=AT, dk=AT, dv=AT, do_sb=256000, do_ss=256, do_sh=64,
                                  dq_sb=256000, dq_ss=256, dq_sh=64, dk_sb=1152, dk_ss=128, dk_sh=64, dv_sb=1152,
                                  dv_ss=128, dv_sh=64)
    assert _capi.lib().hier_cross_attn_bwd(C.addressof(args), None) < 0
    assert says in _capi.lib().hier_last_error().decode()


def test_cross_gradient_entry_refuses_as_many_items_as_a_launch_has_not():
    """512 threads for each key head of 9 keys: 2^32 are refused, less are asked for their workspace."""
    for heads, says in (((1 << 23) - 4, "too many"), ((1 << 23) - 8, "workspace")):
        f = _cross(B=1, Hq=heads, Hk=heads, Sq=1, q_ss=0, k_ss=1 << 22, v_ss=1 << 22)
        wide = {f"{n}_{s}": 64 if s == "sh" else 1 << 30 for n in ("do", "dq", "dk", "dv") for s in ("sb", "ss", "sh")}
        wide.update(do_ss=0)
        args = _capi.HierCrossBwdArgs(f=f, dout=AT, dq=AT, dk=AT, dv=AT, **wide)
        assert _capi.lib().hier_cross_attn_bwd(C.addressof(args), None) < 0
        assert says in _capi.lib().hier_last_error().decode()


def test_entries_refuse_null():
    for name in ("hier_rms_norm", "hier_rms_norm_bwd", "hier_linear", "hier_linear_bwd", "hier_pad_rows", "hier_cross_attn",
                 "hier_cross_attn_bwd"):
        assert getattr(_capi.lib(), name)(None, None) == (_capi.HIER_EINVAL)
    for name in ("hier_rms_norm_bwd_rows", "hier_linear_workspace", "hier_linear_bwd_workspace",
                 "hier_cross_workspace", "hier_cross_bwd_workspace"):
        assert getattr(_capi.lib(), name)(None) == -1


def test_nothing_to_do_is_done():
    for name, args in (("hier_rms_norm", _norm(M=0)), ("hier_linear", _linear(M=0)), ("hier_cross_attn", _cross(B=0)),
                       ("hier_cross_attn", _cross(Sq=0))):
        assert getattr(_capi.lib(), name)(C.addressof(args), None) == 0


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: kernels.rms_norm(x, w[0], eps=1e-6), lambda: kernels.linear_act(x, w),
                 lambda: kernels.cross_attention(q, q, q)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(RuntimeError):
        kernels.linear_act(x.requires_grad_(), w)


def _addresses(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return {t.data_ptr() + t.element_size() * int(i) + b for i in at.flatten() for b in range(t.element_size())}


def test_outputs_over_inputs_are_told():
    """``_share`` against the sets of addresses: a shifted view, a projection's slices, heads
    between heads, gaps, expanded and single rows, other types, and views at random."""
    buf = torch.zeros(3000, dtype=torch.bfloat16)
    rows = buf[:240].view(10, 24)
    qkv = buf[:960].view(2, 10, 3, 2, 8)
    heads = buf[:480].view(10, 2, 3, 8)
    told = [
        (rows[1:], rows[:-1], True), (rows, rows, True), (rows[:5], rows[5:], False),
        (rows[:, :8], rows[:, 8:], False), (rows[:, :9], rows[:, 8:], True), (rows[::2], rows[1::2], False),
        (qkv[:, :, 0], qkv[:, :, 1], False), (qkv[:, :, 1], qkv[:, 1:, 1], True), (qkv[:, :, 1], qkv[:, 1:, 0], False),
        (heads[:, :, 0], heads[:, :, 2], False), (heads[:, 0], heads[:, 1, 1:], False),
        (rows[0, 16:], rows[:, :16], False), (rows[0, 16:], rows[:, :17], True),
        (rows[:1].expand(5, 24), rows[1:], False), (rows[:1].expand(5, 24), rows[:2], True),
        (buf[:100], buf[100:200].view(torch.float32), False), (buf[:102], buf[100:200].view(torch.float32), True),
        (rows[:0], rows, False),
    ]
    for i, (a, b, want) in enumerate(told):
        assert bool(_addresses(a) & _addresses(b)) == want, i
        assert block._share(a, b) == want and block._share(b, a) == want, i
    g = torch.Generator().manual_seed(0)
    pick = lambda *c: c[int(torch.randint(len(c), (), generator=g))]  # noqa: E731
    missed = 0
    for _ in range(3000):
        a, b = (buf.as_strided((pick(1, 2, 3), pick(1, 4, 5), pick(1, 3, 8)), (pick(0, 48, 120), pick(8, 16, 24), 1),
                               pick(0, 1, 3, 8, 16, 24, 40, 200)) for _ in range(2))
        touch = bool(_addresses(a) & _addresses(b))
        assert block._share(a, b) or not touch, (a.stride(), b.stride())
        missed += block._share(a, b) != touch
    assert missed < 600, missed      # (views of unlike pitch that interleave are refused too)


def test_division_of_rows():
    """The magic numbers of a row's query, r / G, for every group of heads up to 300."""
    for g in range(2, 301):
        shift = max(0, math.ceil(math.log2(g)) - 1)
        mul = (1 << (32 + shift)) // g + 1
        assert mul < 1 << 32
        for r in [*range(0, 5 * g), (1 << 30) - 1, (1 << 30) - g, (1 << 30) // g * g, (1 << 30) // g * g - 1]:
            assert (r * mul >> 32) >> shift == r // g, (g, r)


def test_modules_on_the_host():
    """The torch path: parameters, masks, a stream without keys, gates, a kept context."""
    torch.manual_seed(0)
    attn, ffn = CrossAttention(32, 2).double(), FeedForward(32, 64).double()
    assert {k.split(".")[0] for k in attn.state_dict()} == {"q", "k", "v", "o", "norm_q", "norm_k"}
    assert set(ffn.state_dict()) == {"0.weight", "0.bias", "2.weight", "2.bias"}
    x, ctx = torch.randn(3, 6, 32).double(), torch.randn(3, 5, 32).double()
    lens = torch.tensor([5, 2, 0], dtype=torch.int32)
    y = attn(x, ctx, kv_lens=lens)
    assert torch.allclose(y[1:2], attn(x[1:2], ctx[1:2, :2]), atol=1e-5)
    assert torch.allclose(y[2], attn.o.bias.expand(6, 32))
    mask = torch.arange(5) < lens[:, None]
    assert torch.allclose(attn(x, ctx, key_mask=mask), y)
    assert torch.allclose(attn(x, kv=attn.project_context(ctx), kv_lens=lens), y)
    gate = torch.randn(3, 2, 32).double()
    full = gate.repeat_interleave(3, 1)
    assert torch.allclose(attn(x, ctx, kv_lens=lens, residual=x, gate=gate), x + full * y)
    assert torch.allclose(ffn(x, residual=x, gate=gate),
                          x + full * ffn[2](torch.nn.functional.gelu(ffn[0](x), approximate="tanh")))
    with pytest.raises(ValueError):
        attn(x)
    with pytest.raises(ValueError):
        CrossAttention(30, 4)


class _Adapter(torch.nn.Module):
    """A projection with a low-rank term, which shows the projection's weights."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.a = torch.nn.Parameter(torch.randn(2, base.in_features))
        self.b = torch.nn.Parameter(torch.randn(base.out_features, 2))

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + (x @ self.a.to(x.dtype).t()) @ self.b.to(x.dtype).t()


def change_ffn(ffn, how):
    if how == "adapter":
        ffn[0] = _Adapter(ffn[0])
    elif how == "second adapter":
        ffn[2] = _Adapter(ffn[2])
    elif how == "activation":
        ffn[1] = torch.nn.ReLU()
    elif how == "exact gelu":
        ffn[1] = torch.nn.GELU()
    elif how == "appended":
        ffn.append(torch.nn.Tanh())
    elif how == "hook":
        ffn[2].register_forward_hook(lambda m, i, o: 2 * o)
    elif how == "pre-hook":
        ffn[0].register_forward_pre_hook(lambda m, i: (i[0] + 1,))
    elif how == "own forward":
        ffn[0].forward = lambda x: torch.nn.functional.linear(x, ffn[0].weight) - 1


CHANGES = ["adapter", "second adapter", "activation", "exact gelu", "appended", "hook", "pre-hook", "own forward", "none"]


@pytest.mark.parametrize("how", CHANGES)
def test_feed_forward_calls_changed_children(how, monkeypatch):
    """With the kernels' branch open on the host: taken for plain children alone."""
    torch.manual_seed(0)
    ffn = FeedForward(8, 16)
    change_ffn(ffn, how)
    x, res = torch.randn(3, 8), torch.randn(3, 8)
    want = res + torch.nn.Sequential.forward(ffn, x)
    calls = []

    def linear(x, w, b, *, activation=None, residual=None, gate=None):
        calls.append(activation)
        y = torch.nn.functional.linear(x, w, b)
        y = torch.nn.functional.gelu(y, approximate="tanh") if activation else y
        return y if residual is None else residual + y
    monkeypatch.setattr(module, "_block_ok", lambda x, w: True)
    monkeypatch.setattr(module, "linear_act_train", linear)
    assert torch.allclose(ffn(x, residual=res), want, atol=1e-5)
    assert calls == (["gelu_tanh", None] if how == "none" else [])


def test_what_a_plain_child_is():
    p = module._plain
    assert p(torch.nn.Linear(2, 2), torch.nn.Linear) and p(CompatibleLinear(2, 2), torch.nn.Linear, CompatibleLinear)
    assert not p(CompatibleLinear(2, 2), torch.nn.Linear) and not p(torch.nn.LayerNorm(4), RMSNorm)
    hooked = RMSNorm(4)
    assert p(hooked, RMSNorm)
    handle = hooked.register_full_backward_hook(lambda m, i, o: None)
    assert not p(hooked, RMSNorm)
    handle.remove()
    assert p(hooked, RMSNorm)
    weighted = torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(2, 2))
    assert not p(weighted, torch.nn.Linear)
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, i, o: None)
    try:
        assert not p(hooked, RMSNorm)
    finally:
        handle.remove()


@pytest.mark.parametrize("how", ["kv_lens", "key_mask", "both"])
def test_hidden_states_stay_out_on_the_host(how):
    """NaN and infinite padding changes neither values nor gradients, as on the kernels' path."""
    torch.manual_seed(0)
    attn = CrossAttention(32, 2).double()
    x, ctx = torch.randn(3, 6, 32).double().requires_grad_(), torch.randn(3, 5, 32).double()
    lens = torch.tensor([5, 2, 0])
    mask = torch.arange(5) < lens[:, None]
    kw = {"kv_lens": dict(kv_lens=lens), "key_mask": dict(key_mask=mask),
          "both": dict(kv_lens=lens.clamp(min=1), key_mask=mask)}[how]
    k, v = (t.detach() for t in attn.project_context(ctx))
    results = []
    for bad in (0.0, float("nan"), float("inf")):
        kk, vv = k.clone(), v.clone()
        kk[~mask], vv[~mask] = bad, -bad
        kk.requires_grad_(), vv.requires_grad_()
        y = attn(x, kv=(kk, vv), **kw)
        results.append((y, *torch.autograd.grad(y.square().sum(), (x, kk, vv))))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    assert not results[0][2][~mask].any() and not results[0][3][~mask].any()


EPILOGUES = [
    # residual, gate (shape and type; None: none), whether the product's epilogue takes them
    (None, None, True),
    (((2, 6, 8), "same"), None, True),
    (((2, 6, 8), "same"), ((8,), "same"), True),
    (None, ((2, 3, 8), "same"), True),
    (None, ((2, 1, 8), "same"), True),
    (((2, 6, 8), "same"), ((2, 6, 8), "same"), True),
    (((2, 6, 8), "wide"), None, False),
    (((2, 6, 8), "same"), ((2, 3, 8), "wide"), False),
    (((2, 6, 8), "wide"), ((8,), "wide"), False),
    (((1, 6, 8), "same"), None, False),
    (((8,), "same"), None, False),
    (None, ((1, 3, 8), "same"), False),
    (None, ((1, 1, 8), "same"), False),
    (None, ((2, 3, 1), "same"), False),
]


@pytest.mark.parametrize("residual,gate,fits", EPILOGUES)
def test_what_joins_in_the_products_epilogue(residual, gate, fits):
    """What the kernel does not take is applied to its result, as the host's path does."""
    torch.manual_seed(0)
    same, wide = torch.float32, torch.float64
    make = lambda what: None if what is None else torch.randn(what[0], dtype=same if what[1] == "same" else wide)  # noqa: E731
    child, x, res, g = torch.nn.Linear(4, 8), torch.randn(2, 6, 4), make(residual), make(gate)
    calls = []

    def linear(x, w, b, *, residual=None, gate=None):
        calls.append(residual is not None or gate is not None)
        return module._gated(torch.nn.functional.linear(x, w, b), residual, gate)
    got = module._gated_product(linear, x, child, res, g)
    want = module._gated(child(x), res, g)
    assert got.dtype == want.dtype and torch.equal(got, want)
    assert calls == [fits and (res is not None or g is not None)]


def test_gate_rows_have_to_divide():
    for rows, gates in ((5, 2), (1, 3), (4, 0)):
        with pytest.raises(ValueError, match="divide"):
            module._gated(torch.zeros(2, rows, 8), None, torch.zeros(2, gates, 8))
