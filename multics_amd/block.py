"""The rest of a transformer block around the hierarchical attention, on HIP
kernels: a root-mean-square norm with the residual's addition, the matrix
product with bias, activation, gate and residual in its epilogue, and attention
to an encoder's states of another length.  Each comes as a call without
gradient, its gradient, and the two under autograd (``_train``).  Reached as
``multics_amd.kernels.rms_norm`` and so on; ``module.CrossAttention`` and
``module.FeedForward`` run on them.  No counterpart in the reference, which
composes them of torch operations.

Rows are bf16 or fp16, sums fp32.  A backward pass is captured into a graph only
when no eager pass over the same leaves is held any more (outputs or a loss of
it): autograd would join the two passes' streams, which ends the process.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ROWS = torch.contiguous_format          # (empty_like of it: the fastest way to a new tensor)
ACTIVATIONS = {None: 0, "gelu_tanh": 1, "gelu": 2, "silu": 3}

_pack_norm = _capi.packer(_capi.HierRmsNormArgs)
_pack_norm_bwd = _capi.packer(_capi.HierRmsNormBwdArgs)
_pack_linear = _capi.packer(_capi.HierLinearArgs)
_pack_linear_bwd = _capi.packer(_capi.HierLinearBwdArgs)
_pack_pad = _capi.packer(_capi.HierPadRowsArgs)


def _no_grad_call(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} gives no gradient: use {name}_train")


def _gpu_type(name: str, t: torch.Tensor) -> int:
    """The type code of the rows of ``t``, a GPU tensor."""
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
        raise NotImplementedError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if not t.is_cuda:
        raise NotImplementedError(f"{name} must be a GPU tensor")
    return _TYPES[t.dtype]


def _like(name: str, t: torch.Tensor, x: torch.Tensor, shape) -> None:
    if t.shape != tuple(shape) or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must be {x.dtype} {tuple(shape)} on {x.device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _rows(t: torch.Tensor):
    """``t`` [..., C] as rows with contiguous channels (copied if no view of it
    is), and their stride."""
    C = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, C)
    if t.stride(1) != 1 and C > 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else C)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _outs(name: str, out: Optional[torch.Tensor], like: torch.Tensor, shape) -> torch.Tensor:
    """``out`` as given, checked, or a new one."""
    if out is None:
        return like.new_empty(shape)
    _like(name, out, like, shape)
    if not out.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return out


def _operands(x: torch.Tensor, w: torch.Tensor, read=(True, True)):
    """x [..., K] and w [N, K] as a product's operands, 16-byte rows of a multiple of
    eight elements, less than 2^21 apart: their addresses and strides, that multiple, and
    what has to live as long.  Others are copied, with zeros behind (``hier_pad_rows``), if
    the call reads them (``read``)."""
    K = x.shape[-1]
    (x, x_ss), (w, w_ss) = (_rows(t) if r else (t, K) for t, r in zip((x, w), read))
    at = [x.data_ptr(), w.data_ptr()]
    ss = [x_ss, w_ss]
    copy = [r and (K % 8 or s % 8 or p % 16 or not K <= s < 1 << 21) for p, s, r in zip(at, ss, read)]
    Kp = K + -K % 8
    if not any(copy):
        return at[0], x_ss, at[1], w_ss, Kp, (x, w)
    rows = [t.shape[0] if c else 0 for t, c in zip((x, w), copy)]
    buf = x.new_empty((rows[0] + rows[1]) * Kp)
    to = [buf.data_ptr(), buf.data_ptr() + 2 * rows[0] * Kp]
    _capi.call_on(x.device, "hier_pad_rows", _pack_pad(*rows, *ss, *at, *to, K, 0))
    at, ss = zip(*((to[i], Kp) if copy[i] else (at[i], ss[i]) for i in (0, 1)))
    return at[0], ss[0], at[1], ss[1], Kp, (x, w, buf)


def _extent(t: torch.Tensor):
    """The addresses that ``t`` lies within."""
    first, size = t.data_ptr(), t.element_size()
    if t.is_contiguous():
        return first, first + t.numel() * size
    return first, first + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have a byte in common: not where one ends before the other
    begins, nor where both are rows (of whatever inner dimensions) of one pitch that lie
    side by side, as a projection's slices do."""
    (pa, ea), (pb, eb) = _extent(a), _extent(b)
    if ea <= pb or eb <= pa or not a.numel() or not b.numel():
        return False
    (da, ia), (db, ib) = (
        ([(n, s * t.element_size()) for n, s in zip(t.shape, t.stride()) if n > 1 and s], t.element_size())
        for t in (a, b))

    def span(dims, item, below):
        return sum((n - 1) * s for n, s in dims if s < below) + item
    strides = {s for _, s in da + db}
    for least in strides:
        pitch = math.gcd(*(s for s in strides if s >= least))
        at = (pb - pa) % pitch
        if at >= span(da, ia, least) and at + span(db, ib, least) <= pitch:
            return False
    return True


def _apart(name: str, written: torch.Tensor, /, **inputs: Optional[torch.Tensor]) -> None:
    """Refuses an output in the memory of a tensor that is read while it is written."""
    for other, t in inputs.items():
        if t is not None and _share(written, t):
            raise ValueError(f"{name} must not share memory with {other}")


# --------------------------------------------------------------------------
# root-mean-square norm with the residual's addition
# --------------------------------------------------------------------------

def _norm_args(name, x, weight, eps, residual):
    kind = _gpu_type("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have channels, got {tuple(x.shape)}")
    C = x.shape[-1]
    if weight.shape != (C,) or weight.device != x.device or weight.dtype not in _TYPES:
        raise ValueError(f"weight must be [{C}] bf16, fp16 or fp32 on {x.device}, got "
                         f"{tuple(weight.shape)} {weight.dtype} on {weight.device}")
    eps = float(eps)
    if not 0.0 <= eps <= 3.4e38:
        raise ValueError(f"eps must be a number of at least 0, got {eps}")
    if residual is not None:
        _like("residual", residual, x, x.shape)
    return kind, C, eps


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float,
             residual: Optional[torch.Tensor] = None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension of
    ``h = x + residual`` (``hier_rms_norm``); fp32 inside, rounded once.

    ``x`` [..., C] is bf16 or fp16 (C up to 16384), ``weight`` [C] bf16, fp16 or
    fp32.  Returns ``y``, and with ``residual`` (shaped like x) ``(y, h)``; the
    norm is that of the sum before its rounding to ``h``.  No gradient:
    ``rms_norm_train``."""
    _no_grad_call("rms_norm", x, weight, residual)
    return _rms_norm(x, weight, eps, residual)


def _rms_norm(x, weight, eps, residual):
    kind, C, eps = _norm_args("rms_norm", x, weight, eps, residual)
    y = torch.empty_like(x, memory_format=_ROWS)
    h = None if residual is None else torch.empty_like(x, memory_format=_ROWS)
    xr, x_ss = _rows(x)
    r, r_ss = (None, 0) if residual is None else _rows(residual)
    w = weight.contiguous()
    if xr.shape[0]:
        _capi.call_on(x.device, "hier_rms_norm", _pack_norm(
            xr.shape[0], C, eps, kind, _TYPES[w.dtype], xr.data_ptr(), _ptr(r), w.data_ptr(),
            y.data_ptr(), _ptr(h), x_ss, r_ss, C, C))
    return y if h is None else (y, h)


def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *, eps: float,
                      residual: Optional[torch.Tensor] = None, dh: Optional[torch.Tensor] = None):
    """Gradient of ``rms_norm`` (``hier_rms_norm_bwd``) from its inputs and the
    gradients ``dy`` of y and ``dh`` (optional) of h: ``(dx, dweight)``, dx the
    gradient of ``x`` and of ``residual`` alike, dweight fp32 [C], summed in a
    fixed order."""
    kind, C, eps = _norm_args("rms_norm_backward", x, weight, eps, residual)
    _like("dy", dy, x, x.shape)
    if dh is not None:
        _like("dh", dh, x, x.shape)
    dx = torch.empty_like(x, memory_format=_ROWS)
    dw = x.new_empty(C, dtype=torch.float32)
    (xr, x_ss), (g, g_ss) = _rows(x), _rows(dy)
    r, r_ss = (None, 0) if residual is None else _rows(residual)
    d, d_ss = (None, 0) if dh is None else _rows(dh)
    w = weight.contiguous()
    M = xr.shape[0]
    if M == 0:
        return dx, dw.zero_()
    # a row of sums for each workgroup
    rows = _workspace("hier_rms_norm_bwd_rows", _pack_norm_bwd(M, C, eps, kind, 0, *(0,) * 14))
    part = x.new_empty((rows, C), dtype=torch.float32)
    _capi.call_on(x.device, "hier_rms_norm_bwd", _pack_norm_bwd(
        M, C, eps, kind, _TYPES[w.dtype], xr.data_ptr(), _ptr(r), w.data_ptr(), g.data_ptr(), _ptr(d),
        dx.data_ptr(), dw.data_ptr(), part.data_ptr(), x_ss, r_ss, g_ss, d_ss, C, rows))
    return dx, dw


class RMSNormFunction(torch.autograd.Function):
    """Differentiable ``rms_norm``."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, residual)
        ctx.eps = eps
        return _rms_norm(x, weight, eps, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        x, weight, residual = ctx.saved_tensors
        if dy is None and dh is None:
            return None, None, None, None
        if dy is None:                  # h alone was used
            dx, dw = dh, torch.zeros_like(weight)
        else:
            dx, dw = rms_norm_backward(dy, x, weight, eps=ctx.eps, residual=residual, dh=dh)
            dw = dw.to(weight.dtype)
        return dx, dw, None if residual is None else dx, None


def rms_norm_train(x: torch.Tensor, weight: torch.Tensor, *, eps: float,
                   residual: Optional[torch.Tensor] = None):
    """``rms_norm`` under autograd: differentiable in x, weight and residual.
    The same arguments and results."""
    return RMSNormFunction.apply(x, weight, residual, eps)


# --------------------------------------------------------------------------
# matrix product with bias, activation, gate and residual
# --------------------------------------------------------------------------

def _linear_args(x, weight, bias, activation, residual, gate):
    """(type, activation code, M, N, K, rows per gate) of checked arguments."""
    kind = _gpu_type("x", x)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)}, {tuple(weight.shape)}")
    N, K = weight.shape
    _like("weight", weight, x, (N, K))
    if bias is not None:
        _like("bias", bias, x, (N,))
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(map(repr, ACTIVATIONS))}")
    M = x.numel() // K
    if residual is not None:
        _like("residual", residual, x, (*x.shape[:-1], N))
    per = 1
    if gate is not None:
        if gate.dim() != x.dim() and gate.dim() != 1:
            raise ValueError(f"gate must be [..., F, N] or [N], got {tuple(gate.shape)}")
        lead, rows = (x.shape[:-2], x.shape[-2]) if x.dim() > 1 else ((), 1)
        if gate.dim() == 1:
            _like("gate", gate, x, (N,))
            per = max(M, 1)
        else:
            F = gate.shape[-2]
            _like("gate", gate, x, (*lead, F, N))
            if F < 1 or rows % F:
                raise ValueError(f"{rows} rows do not divide into {F} gate rows")
            per = max(rows // F, 1)
    return kind, ACTIVATIONS[activation], M, N, K, per


def _workspace(name: str, args: bytes) -> int:
    size = getattr(_capi.lib(), name)(args)
    if size < 0:
        _capi.check(_capi.HIER_EINVAL, name)
    return size


def _linear(x, weight, bias, activation, residual, gate, out, preact):
    kind, act, M, N, K, per = _linear_args(x, weight, bias, activation, residual, gate)
    shape = (*x.shape[:-1], N)
    given = out is not None
    out = _outs("out", out, x, shape)
    if given:
        same = residual is not None and residual.data_ptr() == out.data_ptr() and residual.is_contiguous()
        _apart("out", out, x=x, weight=weight, bias=bias, gate=gate, residual=None if same else residual)
    if M == 0:
        return out
    x_at, x_ss, w_at, w_ss, K, kept = _operands(x, weight)
    b = None if bias is None else bias.contiguous()
    r, r_ss = (None, 0) if residual is None else _rows(residual)
    g, g_ss = (None, 0) if gate is None else _rows(gate)
    fields = (M, N, K, kind, act, x_at, w_at, _ptr(b), _ptr(r), _ptr(g), out.data_ptr(),
              _ptr(preact), x_ss, w_ss, r_ss, g_ss, N, N, per)
    size = 0 if M <= 8 else _workspace("hier_linear_workspace", _pack_linear(*fields, 0, 0))
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _capi.call_on(x.device, "hier_linear", _pack_linear(*fields, _ptr(ws), size))
    return out


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
               activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + gate * act(x @ weight.T + bias)`` in one pass
    (``hier_linear``); fp32 inside, rounded once.

    ``x`` [..., K] and ``weight`` [N, K] are bf16 or fp16; ``activation`` is None,
    ``"gelu_tanh"``, ``"gelu"`` or ``"silu"``.  ``residual`` is [..., N]; ``gate`` is
    [N], or [..., F, N] whose rows scale S / F rows of x's S each (a frame's tokens
    share their frame's gate, as in ``gated_residual``).  ``out`` (optional, contiguous)
    may be ``residual`` itself and shares no memory with the inputs otherwise.  Rows of a
    multiple of eight channels are read in place, others, and rows 2^21 elements apart or
    more, are copied with zeros behind.  No gradient: ``linear_act_train``."""
    _no_grad_call("linear_act", x, weight, bias, residual, gate)
    return _linear(x, weight, bias, activation, residual, gate, out, None)


def linear_act_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *,
                        preact: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                        gate: Optional[torch.Tensor] = None, need=("x", "weight", "bias", "gate")) -> dict:
    """Gradients of ``linear_act`` (``hier_linear_bwd``) from the gradient ``dy``
    [..., N] of its output and ``preact`` [..., N], the values before the activation
    (not needed without an activation and the gate's gradient): those of ``need``,
    by name, in x's type.  The residual's gradient is ``dy``.  Sums are taken in a
    fixed order: equal inputs give equal bits."""
    kind, act, M, N, K, per = _linear_args(x, weight, None, activation, None, gate)
    shape = (*x.shape[:-1], N)
    _like("dy", dy, x, shape)
    need = [n for n in need if n != "gate" or gate is not None]
    if preact is None and (act or "gate" in need):
        raise ValueError("linear_act_backward needs preact, the values before the activation")
    if preact is not None:
        _like("preact", preact, x, shape)
    new = lambda *s: x.new_empty(s)  # noqa: E731
    if M == 0:
        made = {"x": lambda: torch.zeros_like(x), "weight": lambda: torch.zeros_like(weight),
                "bias": lambda: new(N).zero_(), "gate": lambda: torch.zeros_like(gate)}
        return {n: made[n]() for n in need}
    x_at, x_ss, w_at, w_ss, Kp, kept = _operands(x, weight, ("weight" in need, "x" in need))
    g_dy, dy_ss = _rows(dy)
    if not act and gate is None:
        preact = None
    z, z_ss = (None, 0) if preact is None else _rows(preact)
    g, g_ss = (None, 0) if gate is None else _rows(gate)
    dx = new(M, Kp) if "x" in need else None
    dw = new(N, Kp) if "weight" in need else None
    db = new(N) if "bias" in need else None
    dg = new(M // per, N) if "gate" in need else None
    fields = (M, N, Kp, kind, act, x_at, w_at, _ptr(g), g_dy.data_ptr(), _ptr(z), _ptr(dx),
              _ptr(dw), _ptr(db), _ptr(dg), x_ss, w_ss, g_ss, dy_ss, z_ss, Kp, Kp, per)
    size = _workspace("hier_linear_bwd_workspace", _pack_linear_bwd(*fields, 0, 0))
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _capi.call_on(x.device, "hier_linear_bwd", _pack_linear_bwd(*fields, _ptr(ws), size))
    made = {"x": lambda: (dx if Kp == K else dx[:, :K]).reshape(x.shape),
            "weight": lambda: dw if Kp == K else dw[:, :K],
            "bias": lambda: db,
            "gate": lambda: dg.reshape(gate.shape)}
    return {n: made[n]() for n in need}


class LinearActFunction(torch.autograd.Function):
    """Differentiable ``linear_act``: keeps x, the weights, the gate and, with an
    activation or a gate, the values before the activation in x's type."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, activation):
        keep = any(ctx.needs_input_grad) and (activation is not None or
                                              gate is not None and ctx.needs_input_grad[4])
        z = x.new_empty((*x.shape[:-1], weight.shape[0])) if keep else None
        y = _linear(x, weight, bias, activation, residual, gate, None, z)
        ctx.save_for_backward(x, weight, gate, z)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, gate, z = ctx.saved_tensors
        names = ("x", "weight", "bias", "residual", "gate")
        want = [n for n, w in zip(names, ctx.needs_input_grad) if w]
        need = [n for n in want if n != "residual"]
        got = linear_act_backward(dy, x, weight, preact=z, activation=ctx.activation, gate=gate,
                                  need=need) if need else {}
        if "residual" in want:
            got["residual"] = dy
        return *(got.get(n) for n in names), None


def linear_act_train(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                     gate: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear_act`` under autograd: differentiable in every tensor.  The same
    arguments and results."""
    return LinearActFunction.apply(x, weight, bias, residual, gate, activation)


# --------------------------------------------------------------------------
# attention to an encoder's states
# --------------------------------------------------------------------------

_pack_cross = _capi.packer(_capi.HierCrossArgs)
_pack_cross_bwd = _capi.packer(_capi.HierCrossBwdArgs)


def _heads(t: torch.Tensor):
    """``t`` [B, S, H, D] readable in 16-byte rows (copied if it is not), and its
    strides over streams, tokens and heads (0 over one alone)."""
    B, S, H, D = t.shape
    for _ in range(2):
        sb, ss, sh, unit = t.stride()
        sb, ss, sh = sb if B > 1 else 0, ss if S > 1 else 0, sh if H > 1 else 0
        if unit == 1 and sb % 8 == 0 and ss % 8 == 0 and sh % 8 == 0 and t.data_ptr() % 16 == 0 and \
                (ss >= D or S < 2) and 65 * ss + H * sh < 1 << 30:
            break
        t = _capi.aligned(t)
    return t, (sb, ss, sh)


def _cross_args(q, k, v, kv_lens, key_mask, scale):
    """Checked arguments of the cross attention: (sizes and scale, q, k, v with their strides, lens,
    mask)."""
    kind = _gpu_type("q", q)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [B, S, H, D], got {tuple(t.shape)}")
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    _like("k", k, q, (B, Sk, Hk, D))
    _like("v", v, q, (B, Sk, Hk, D))
    if D not in (64, 128):
        raise NotImplementedError(f"cross attention supports head_dim 64/128, got {D}")
    if Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are not a multiple of {Hk} key heads")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"the softmax scale must be positive, got {scale}")
    if kv_lens is not None:
        if kv_lens.shape != (B,) or kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.device != q.device:
            raise ValueError(f"kv_lens must be int32 [{B}] on {q.device}, got {kv_lens.dtype} "
                             f"{tuple(kv_lens.shape)} on {kv_lens.device}")
        if kv_lens.dtype == torch.int64:
            kv_lens = kv_lens.clamp(0, Sk).to(torch.int32)
        kv_lens = kv_lens.contiguous()
    if key_mask is not None:
        if key_mask.shape != (B, Sk) or key_mask.dtype != torch.bool or key_mask.device != q.device:
            raise ValueError(f"key_mask must be bool {(B, Sk)} on {q.device}, got {key_mask.dtype} "
                             f"{tuple(key_mask.shape)} on {key_mask.device}")
        if key_mask.stride(1) != 1 and Sk > 1:
            key_mask = key_mask.contiguous()
    return (B, Hq, Hk, D, kind, scale, Sq, Sk), _heads(q), _heads(k), _heads(v), kv_lens, key_mask


def _cross_fields(sizes, q, k, v, o, lse, lens, mask):
    (qt, qs), (kt, ks), (vt, vs), (ot, os) = q, k, v, o
    return (*sizes, qt.data_ptr(), kt.data_ptr(), vt.data_ptr(), ot.data_ptr(), _ptr(lse), _ptr(lens), _ptr(mask),
            *qs, *ks, *vs, *os, 0 if mask is None else mask.stride(0))


def _check_lse(lse, sizes, device):
    B, Hq, _, _, _, _, Sq, _ = sizes
    if lse.shape != (B, Hq, Sq) or lse.dtype != torch.float32 or lse.device != device or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous fp32 {(B, Hq, Sq)} on {device}, got {lse.dtype} "
                         f"{tuple(lse.shape)} on {lse.device}")


def _cross(q, k, v, kv_lens, key_mask, scale, out, lse):
    sizes, qh, kh, vh, lens, mask = _cross_args(q, k, v, kv_lens, key_mask, scale)
    if out is None:
        out = torch.empty_like(q, memory_format=_ROWS)
    else:
        _like("out", out, q, q.shape)
        _apart("out", out, q=q, k=k, v=v, kv_lens=kv_lens, key_mask=key_mask)
    oh = _heads(out)
    B, Hq, _, D, _, _, Sq, _ = sizes
    if oh[0] is not out or any(n > 1 and s < D for n, s in zip((B, Sq, Hq), oh[1])):
        raise ValueError("out must have rows of its own, a unit-stride head dimension and 16-byte rows")
    if lse is not None:
        _check_lse(lse, sizes, q.device)
    if B == 0 or Sq == 0:
        return out
    fields = _cross_fields(sizes, qh, kh, vh, oh, lse, lens, mask)
    size = _workspace("hier_cross_workspace", _pack_cross(*fields, 0, 0))
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _capi.call_on(q.device, "hier_cross_attn", _pack_cross(*fields, _ptr(ws), size))
    return out


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` over another sequence's keys (``hier_cross_attn``).

    ``q`` [B, Sq, H, D] and ``k`` / ``v`` [B, Sk, Hk, D] are bf16 or fp16 views
    (unit-stride channels, D 64 or 128; others are copied), H a multiple of Hk:
    query heads i * H/Hk .. share key head i.  A stream's keys are the first
    ``kv_lens[b]`` (int32 [B] on the GPU, taken within [0, Sk]) whose ``key_mask``
    [B, Sk] (bool) is true; what else k and v hold is not read.  Returns [B, Sq, H, D]
    (``out`` where given); a row that sees no key is 0.  ``lse`` (optional, contiguous
    fp32 [B, H, Sq]) receives the natural-log softmax normaliser, -inf for such a
    row.  ``out`` and ``lse`` share no memory with the inputs or one another.  Sq may be
    one token: the keys are then cut into parts that fill the GPU.  No gradient: ``cross_attention_train``."""
    _no_grad_call("cross_attention", q, k, v)
    if lse is not None:
        _apart("lse", lse, q=q, k=k, v=v, kv_lens=kv_lens, key_mask=key_mask, out=out)
    return _cross(q, k, v, kv_lens, key_mask, scale, out, lse)


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             out: torch.Tensor, lse: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                             key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None):
    """Gradients ``(dq, dk, dv)`` of ``cross_attention`` (``hier_cross_attn_bwd``) from its
    inputs, its ``out`` and ``lse`` and the gradient ``dout`` of out; bf16.  dk and dv are
    summed over the query heads that share a head and 0 for keys that are not seen.
    Sums are taken in a fixed order: equal inputs give equal bits."""
    sizes, qh, kh, vh, lens, mask = _cross_args(q, k, v, kv_lens, key_mask, scale)
    if q.dtype != torch.bfloat16:
        raise NotImplementedError(f"cross attention's gradients are bf16 only, got {q.dtype}")
    _like("out", out, q, q.shape)
    _like("dout", dout, q, q.shape)
    _check_lse(lse, sizes, q.device)
    B, _, _, _, _, _, Sq, Sk = sizes
    dq, dk, dv = (torch.empty_like(t, memory_format=_ROWS) for t in (q, k, v))
    if B == 0 or Sq == 0 or Sk == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    oh, (dot, dos) = _heads(out), _heads(dout)
    fields = _cross_fields(sizes, qh, kh, vh, oh, lse, lens, mask)
    size = _workspace("hier_cross_bwd_workspace", _pack_cross(*fields, 0, 0))
    ws = q.new_empty(size, dtype=torch.uint8)
    strides = lambda t: t.stride()[:3]  # noqa: E731
    _capi.call_on(q.device, "hier_cross_attn_bwd", _pack_cross_bwd(
        *fields, ws.data_ptr(), size, dot.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dos,
        *strides(dq), *strides(dk), *strides(dv)))
    return dq, dk, dv


class CrossAttentionFunction(torch.autograd.Function):
    """Differentiable ``cross_attention``."""

    @staticmethod
    def forward(ctx, q, k, v, kv_lens, key_mask, scale):
        if q.dtype != torch.bfloat16 and any(ctx.needs_input_grad):
            raise NotImplementedError(f"cross attention's gradients are bf16 only, got {q.dtype}")
        if q.dim() != 4:
            raise ValueError(f"q must be [B, S, H, D], got {tuple(q.shape)}")
        B, Sq, H, _ = q.shape
        lse = q.new_empty((B, H, Sq), dtype=torch.float32)
        out = _cross(q, k, v, kv_lens, key_mask, scale, None, lse)
        ctx.save_for_backward(q, k, v, out, lse, kv_lens, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lens, key_mask = ctx.saved_tensors
        grads = cross_attention_backward(dout, q, k, v, out, lse, kv_lens=kv_lens, key_mask=key_mask,
                                         scale=ctx.scale)
        return *grads, None, None, None


def cross_attention_train(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                          kv_lens: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """``cross_attention`` under autograd: differentiable in q, k and v (bf16)."""
    return CrossAttentionFunction.apply(q, k, v, kv_lens, key_mask, scale)
