"""Speed and exactness of the rest of a transformer block around the hierarchical attention.

* ``norm`` / ``norm_grad``: root-mean-square norm over the model's channels, with the addition of a
  residual before it (``kernels.rms_norm`` / ``rms_norm_train``).
* ``linear`` / ``linear_grad``: matrix product with bias, activation, gate and residual in its epilogue,
  and the training step of it (``kernels.linear_act`` / ``linear_act_train``).
* ``cross`` / ``cross_grad``: attention to an encoder's states of another length, with contexts of
  unlike lengths or with masked keys, and its training step (``kernels.cross_attention`` /
  ``cross_attention_train``).

``run`` computes each in elementary torch operations in 32 bits, or, where ``own`` is set, calls the
framework.  ``exact`` gives the same outputs in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------


def listed():
    return [
        # one denoised token for each of two players: what counts is the launch
        dict(name="norm_token", op="norm", M=2, C=1536, dtype="bf16", residual=False),
        # the four-player clip's residual stream, added to and normed
        dict(name="norm_clip", op="norm", M=18816, C=1536, dtype="bf16", residual=True),
        # the same in a training step
        dict(name="norm_grad_clip", op="norm_grad", M=18816, C=1536, dtype="bf16", residual=True),
        # a single token through the first product of a feed-forward: the weights are what is read
        dict(name="linear_token", op="linear", M=1, K=1536, N=8960, act="gelu_tanh", dtype="bf16",
             residual=False, gates=0),
        # a handful of rows, sizes that fill no tile, 16-bit floats
        dict(name="linear_odd", op="linear", M=77, K=1000, N=1811, act="silu", dtype="fp16",
             residual=True, gates=0),
        # the four-player clip through the first product of its feed-forward
        dict(name="linear_up", op="linear", M=18816, K=1536, N=8960, act="gelu_tanh", dtype="bf16",
             residual=False, gates=0),
        # a ten-player rollout block (3 frames of 220 tokens each) through the second one, gated for
        # each player's frame and added to the residual stream
        dict(name="linear_down", op="linear", M=6600, K=8960, N=1536, act="none", dtype="bf16",
             residual=True, gates=30),
        # the training step of a feed-forward's first product
        dict(name="linear_grad_up", op="linear_grad", M=9408, K=1536, N=8960, act="gelu_tanh",
             dtype="bf16", residual=False, gates=0),
        # one token for each of four streams against long contexts, shared key heads
        dict(name="cross_token", op="cross", B=4, Sq=1, Sk=4096, Hq=32, Hk=8, D=128, dtype="bf16",
             keys="lens"),
        # the ten-player rollout block against each player's text states
        dict(name="cross_block", op="cross", B=10, Sq=660, Sk=512, Hq=12, Hk=12, D=128, dtype="bf16",
             keys="lens"),
        # the training step of the four-player clip against its text states
        dict(name="cross_grad_clip", op="cross_grad", B=4, Sq=4620, Sk=512, Hq=12, Hk=12, D=128,
             dtype="bf16", keys="all"),
        # odd lengths, shared key heads, masked keys, a stream whose mask leaves nothing
        dict(name="cross_grad_odd", op="cross_grad", B=3, Sq=257, Sk=77, Hq=10, Hk=5, D=64,
             dtype="bf16", keys="mask"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear", "linear_grad", "cross", "cross", "cross_grad"])
    dtype = "bf16" if op.endswith("grad") else rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm", "norm_grad"):
        C = rng.choice([_spread(rng, 64, 5120), 8 * _spread(rng, 8, 640)])
        return dict(op=op, M=_spread(rng, 1, min(18816, 28000000 // C)), C=C, dtype=dtype,
                    residual=rng.random() < 0.5)
    if op in ("linear", "linear_grad"):
        M = _spread(rng, 1, 18816 if op == "linear" else 9408)
        K, N = (rng.choice([8 * _spread(rng, 8, 1120), _spread(rng, 64, 9000)]) for _ in range(2))
        while M * K * N > 125000000000:
            K, N = max(64, K // 2), max(64, N // 2)
        act = rng.choice(["none", "gelu_tanh", "gelu", "silu"])
        gates = rng.choice([0, 0, 1, 3, 10])
        residual = rng.random() < 0.5 or gates > 0
        if gates:
            M = -(-M // gates) * gates
        return dict(op=op, M=M, K=K, N=N, act=act, dtype=dtype, residual=residual, gates=gates)
    Hk, G = rng.choice([(12, 1), (8, 1), (5, 1), (16, 1), (4, 4), (2, 6), (8, 4), (1, 8)])
    B, D = rng.randint(1, 6), rng.choice([64, 128])
    Sk = _spread(rng, 1, 8192)
    Sq = rng.choice([1, _spread(rng, 1, 5000), _spread(rng, 1, 5000)])
    while B * Sq * Sk * Hk * G > 4 * 4620 * 512 * 12:
        Sk, Sq = max(1, Sk // 2), max(1, Sq * 2 // 3)
    return dict(op=op, B=B, Sq=Sq, Sk=Sk, Hq=Hk * G, Hk=Hk, D=D, dtype=dtype,
                keys=rng.choice(["all", "lens", "lens", "mask"]))


def _lens(c):
    """The keys of each stream that hold a token: from all of them down to a seventh, for the last of
    three streams or more none."""
    B, Sk = c["B"], c["Sk"]
    if c["keys"] == "all":
        return [Sk] * B
    lens = [max(1, Sk - (Sk * 6 * b) // (7 * B)) for b in range(B)]
    if B >= 3 and c["keys"] == "mask":
        lens[-1] = 0
    return lens


def work(case):
    c = case
    if c["op"] == "norm":
        t = c["M"] * c["C"]
        return {"bytes": 2 * t * (4 if c["residual"] else 2) + 4 * c["C"], "flops": 5 * t}
    if c["op"] == "norm_grad":
        # forward, then the gradients of the output and of the sum in, the gradient of both addends out
        t = c["M"] * c["C"]
        return {"bytes": 2 * t * (7 if c["residual"] else 4) + 8 * c["C"], "flops": 16 * t}
    if c["op"] in ("linear", "linear_grad"):
        M, K, N = c["M"], c["K"], c["N"]
        io = M * K + N * K + N + M * N * (2 if c["residual"] else 1) + c["gates"] * N
        if c["op"] == "linear":
            return {"bytes": 2 * io, "flops": 2 * M * N * K}
        back = M * N + M * K + N * K + N + c["gates"] * N      # the output's gradient in, the others out
        return {"bytes": 2 * (io + back), "flops": 6 * M * N * K}
    seen = sum(_lens(c))
    q, kv = c["B"] * c["Sq"] * c["Hq"] * c["D"], 2 * seen * c["Hk"] * c["D"]
    flops = 4 * c["Sq"] * seen * c["Hq"] * c["D"]
    if c["op"] == "cross":
        return {"bytes": 2 * (2 * q + kv), "flops": flops}
    whole = 2 * c["B"] * c["Sk"] * c["Hk"] * c["D"]
    return {"bytes": 2 * (4 * q + kv + whole), "flops": 7 * flops // 2}


# ---- inputs ------------------------------------------------------------------------------------


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _generator(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=_device())


def _stream(g, rows, channels):
    """Rows of a residual stream: channels of unlike size, tokens of unlike size."""
    return _normal(g, rows, channels) * torch.exp(0.5 * _normal(g, 1, channels)) * \
        torch.exp(0.3 * _normal(g, rows, 1))


def _norm_inputs(c, seed):
    g, dt = _generator(seed), TYPES[c["dtype"]]
    M, C = c["M"], c["C"]
    st = dict(case=c, x=_stream(g, M, C).to(dt), w=1 + 0.2 * _normal(g, C))
    if c["residual"]:
        st["r"] = (2 * _stream(g, M, C)).to(dt)
    if c["op"] == "norm_grad":
        st["dy"] = (0.1 * _normal(g, M, C)).to(dt)
        if c["residual"]:
            st["dh"] = (0.1 * _normal(g, M, C)).to(dt)
        if own:
            for name in ("x", "w", "r"):
                if name in st:
                    st[name].requires_grad_()
    return st


def _linear_inputs(c, seed):
    g, dt = _generator(seed), TYPES[c["dtype"]]
    M, K, N = c["M"], c["K"], c["N"]
    st = dict(case=c, x=(_normal(g, M, K) * torch.exp(0.3 * _normal(g, 1, K))).to(dt),
              w=(_normal(g, N, K) / math.sqrt(K)).to(dt), b=(0.3 * _normal(g, N)).to(dt))
    if c["residual"]:
        st["r"] = (2 * _normal(g, M, N)).to(dt)
    if c["gates"]:
        st["gate"] = (0.5 * _normal(g, c["gates"], N)).to(dt)
    if c["op"] == "linear_grad":
        st["dy"] = (0.1 * _normal(g, M, N)).to(dt)
        if own:
            for name in ("x", "w", "b", "r", "gate"):
                if name in st:
                    st[name].requires_grad_()
    return st


def _cross_inputs(c, seed):
    """Normed queries and keys, values, and which keys hold a token; the rest hold zeros."""
    g, dt, dev = _generator(seed), TYPES[c["dtype"]], _device()
    B, Sq, Sk, D = c["B"], c["Sq"], c["Sk"], c["D"]
    q = _normal(g, B, Sq, c["Hq"], D) * torch.exp(0.3 * _normal(g, 1, 1, 1, D))
    k = _normal(g, B, Sk, c["Hk"], D) * torch.exp(0.3 * _normal(g, 1, 1, 1, D))
    v = _normal(g, B, Sk, c["Hk"], D) * torch.exp(0.3 * _normal(g, B, Sk, 1, 1))
    st = dict(case=c)
    seen = torch.ones(B, Sk, dtype=torch.bool, device=dev)
    if c["keys"] != "all":
        lens = torch.tensor(_lens(c), dtype=torch.int32, device=dev)
        seen = torch.arange(Sk, device=dev)[None] < lens[:, None]
        if c["keys"] == "lens":
            st["lens"] = lens
        else:       # as many keys of each stream, anywhere
            order = torch.rand(B, Sk, generator=g, device=dev).argsort(1)
            seen = torch.zeros_like(seen).scatter_(1, order, seen)
            st["mask"] = seen
    st.update(q=q.to(dt), k=(k * seen[:, :, None, None]).to(dt), v=(v * seen[:, :, None, None]).to(dt))
    if c["op"] == "cross_grad":
        st["dout"] = (0.1 * _normal(g, B, Sq, c["Hq"], D)).to(dt)
        if own:
            for name in ("q", "k", "v"):
                st[name].requires_grad_()
    return st


def prepare(case, seed):
    make = {"norm": _norm_inputs, "norm_grad": _norm_inputs, "linear": _linear_inputs,
            "linear_grad": _linear_inputs, "cross": _cross_inputs, "cross_grad": _cross_inputs}
    return make[case["op"]](case, seed)


# ---- the operators -----------------------------------------------------------------------------


def _norm(st):
    c, r = st["case"], st.get("r")
    if own:
        from multics_amd import kernels
        return kernels.rms_norm(st["x"], st["w"], eps=EPS, residual=r)
    dt = st["x"].dtype
    h = st["x"].float()
    if r is not None:
        h = h + r.float()
    y = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * st["w"]).to(dt)
    return (y, h.to(dt)) if c["residual"] else y


def _norm_grad(st):
    c, x, w, dy, r, dh = st["case"], st["x"], st["w"], st["dy"], st.get("r"), st.get("dh")
    if own:
        from multics_amd import kernels
        if r is None:
            y = kernels.rms_norm_train(x, w, eps=EPS)
            return y, *torch.autograd.grad(y, (x, w), dy)
        y, h = kernels.rms_norm_train(x, w, eps=EPS, residual=r)
        return y, h, *torch.autograd.grad((y, h), (x, w, r), (dy, dh))
    dt = x.dtype
    h = x.float() if r is None else x.float() + r.float()
    s = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    xh, g = h * s, dy.float()
    y = (xh * w).to(dt)
    gw = g * w
    dx = s * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    dw = (g * xh).sum(0)
    if r is None:
        return y, dx.to(dt), dw
    dx = (dx + dh.float()).to(dt)
    return y, h.to(dt), dx, dw, dx


def _act(z, kind):
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, kind):
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _own_kind(c):
    return None if c["act"] == "none" else c["act"]


def _rows(gate, M):
    """The gate of each of M rows."""
    return gate.repeat_interleave(M // gate.shape[0], 0)


def _linear(st):
    c, r, gate = st["case"], st.get("r"), st.get("gate")
    if own:
        from multics_amd import kernels
        return kernels.linear_act(st["x"], st["w"], st["b"], activation=_own_kind(c), residual=r, gate=gate)
    y = _act(torch.matmul(st["x"].float(), st["w"].float().t()) + st["b"].float(), c["act"])
    if gate is not None:
        y = y * _rows(gate.float(), c["M"])
    if r is not None:
        y = r.float() + y
    return y.to(st["x"].dtype)


def _linear_grad(st):
    c, x, w, b, dy, r, gate = (st["case"], st["x"], st["w"], st["b"], st["dy"], st.get("r"), st.get("gate"))
    if own:
        from multics_amd import kernels
        y = kernels.linear_act_train(x, w, b, activation=_own_kind(c), residual=r, gate=gate)
        leaves = [t for t in (x, w, b, gate) if t is not None]
        return y, *torch.autograd.grad(y, leaves, dy)
    return _linear_grad_form(c, x, w, b, dy, r, gate, torch.float32, x.dtype)


def _linear_grad_form(c, x, w, b, dy, r, gate, wide, dt):
    M, xf, wf, g = c["M"], x.to(wide), w.to(wide), dy.to(wide)
    z = torch.matmul(xf, wf.t()) + b.to(wide)
    a = _act(z, c["act"])
    rows = None if gate is None else _rows(gate.to(wide), M)
    y = a if rows is None else a * rows
    y = y if r is None else r.to(wide) + y
    dz = (g if rows is None else g * rows) * _act_grad(z, c["act"])
    out = [y.to(dt), torch.matmul(dz, wf).to(dt), torch.matmul(dz.t(), xf).to(dt), dz.sum(0).to(dt)]
    if gate is not None:
        out.append((g * a).reshape(gate.shape[0], -1, c["N"]).sum(1).to(dt))
    return tuple(out)


def _cross_parts(st, wide):
    """Head-major queries, keys and values in `wide`, key heads repeated for the query heads that share
    them, and the seen keys as [B, 1, 1, Sk]."""
    c = st["case"]
    G = c["Hq"] // c["Hk"]
    q = st["q"].detach().to(wide).transpose(1, 2).contiguous()
    k, v = (st[n].detach().to(wide).transpose(1, 2).repeat_interleave(G, 1).contiguous() for n in ("k", "v"))
    if "lens" in st:
        seen = torch.arange(c["Sk"], device=q.device)[None] < st["lens"][:, None]
    else:
        seen = st.get("mask")
    return q, k, v, None if seen is None else seen[:, None, None]


def _softmax(q, k, seen, D):
    s = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)
    if seen is not None:
        s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > float("-inf"), m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _cross(st):
    if own:
        from multics_amd import kernels
        return kernels.cross_attention(st["q"], st["k"], st["v"], kv_lens=st.get("lens"),
                                       key_mask=st.get("mask"))
    q, k, v, seen = _cross_parts(st, torch.float32)
    p = _softmax(q, k, seen, st["case"]["D"])
    return torch.matmul(p, v).transpose(1, 2).to(st["q"].dtype)


def _cross_grad(st):
    if own:
        from multics_amd import kernels
        out = kernels.cross_attention_train(st["q"], st["k"], st["v"], kv_lens=st.get("lens"),
                                            key_mask=st.get("mask"))
        return out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
    return _cross_grad_form(st, torch.float32, st["q"].dtype)


def _cross_grad_form(st, wide, dt):
    c = st["case"]
    q, k, v, seen = _cross_parts(st, wide)
    do = st["dout"].to(wide).transpose(1, 2).contiguous()
    p = _softmax(q, k, seen, c["D"])
    out = torch.matmul(p, v)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) / math.sqrt(c["D"])
    shared = lambda t: t.reshape(c["B"], c["Hk"], -1, c["Sk"], c["D"]).sum(2)  # noqa: E731
    dk = shared(torch.matmul(ds.transpose(2, 3), q))
    dv = shared(torch.matmul(p.transpose(2, 3), do))
    return tuple(t.transpose(1, 2).to(dt) for t in (out, torch.matmul(ds, k), dk, dv))


def run(state):
    call = {"norm": _norm, "norm_grad": _norm_grad, "linear": _linear, "linear_grad": _linear_grad,
            "cross": _cross, "cross_grad": _cross_grad}
    return call[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_norm(c, st):
    h = st["x"].detach().double()
    if c["residual"]:
        h = h + st["r"].detach().double()
    rms = torch.sqrt(h.square().sum(-1, keepdim=True) / c["C"] + EPS)
    w = st["w"].detach().double()
    y = h / rms * w
    if c["op"] == "norm":
        return (y, h) if c["residual"] else y
    dy = st["dy"].double()
    inner = (dy * w * h).sum(-1, keepdim=True)
    dx = dy * w / rms - h * inner / (c["C"] * rms ** 3)
    dw = (dy * h / rms).sum(0)
    if not c["residual"]:
        return y, dx, dw
    dx = dx + st["dh"].double()
    return y, h, dx, dw, dx


def _wide_act(z, kind):
    """(value, slope)."""
    if kind == "gelu_tanh":
        a, b = 0.7978845608028654, 0.044715
        s = torch.sigmoid(2 * a * (z + b * z * z * z))
        return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * b * z * z)
    if kind == "gelu":
        s = torch.special.ndtr(z)
        return z * s, s + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def _exact_linear(c, st):
    x, w, b = (st[n].detach().double() for n in ("x", "w", "b"))
    z = torch.addmm(b, x, w.t())
    a, slope = _wide_act(z, c["act"])
    G = max(1, c["gates"])
    gate = st["gate"].detach().double()[:, None] if c["gates"] else torch.ones((), device=x.device).double()
    split = lambda t: t.reshape(G, c["M"] // G, -1)  # noqa: E731
    y = (split(a) * gate).reshape(c["M"], -1)
    if c["residual"]:
        y = y + st["r"].detach().double()
    if c["op"] == "linear":
        return y
    dy = st["dy"].double()
    dz = (split(dy) * gate).reshape(c["M"], -1) * slope
    out = (y, dz @ w, dz.t() @ x, dz.sum(0))
    return out + ((split(dy) * split(a)).sum(1),) if c["gates"] else out


def _exact_cross(c, st):
    """A stream at a time, over the keys that it sees alone."""
    B, Sq, Sk, Hq, Hk, D = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D"))
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    grad = c["op"] == "cross_grad"
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        if "mask" in st:
            at = st["mask"][b].nonzero()[:, 0]
        else:
            at = torch.arange(_lens(c)[b], device=q.device)
        if at.numel() == 0:
            continue
        for h in range(Hq):
            kh = h // (Hq // Hk)
            K, V, Q = k[b, at, kh], v[b, at, kh], q[b, :, h]
            P = torch.softmax(Q @ K.t() * D ** -0.5, -1)
            out[b, :, h] = P @ V
            if grad:
                dO = st["dout"][b, :, h].double()
                dP = dO @ V.t()
                dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * D ** -0.5
                dq[b, :, h] = dS @ K
                dk[b, at, kh] += dS.t() @ Q
                dv[b, at, kh] += P.t() @ dO
    return (out, dq, dk, dv) if grad else out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op.startswith("norm"):
        return _exact_norm(case, st)
    return _exact_linear(case, st) if op.startswith("linear") else _exact_cross(case, st)
