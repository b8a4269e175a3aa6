"""Speed and exactness of three operators of a rollout with per-head norms and an 8-bit KV cache.

* ``norm`` / ``norm_grad``: RMSNorm of queries and keys for each head and the position rotation, in one
  pass, and its gradient (``kernels.qk_head_prologue`` / ``qk_head_prologue_backward``).
* ``append``: a block's keys and values into the pages of a paged cache held in 8 bits (e4m3), with one
  power-of-two scale for 16 tokens and a head (``HierPagedKVCache(dtype=torch.float8_e4m3fn)``).
* ``attend``: the hierarchical attention of a rollout block over that cache
  (``kernels.hier_cached_attention_fp8``).

``run`` computes each in elementary torch operations in 32 bits, or, where ``own`` is set, calls the
framework.  ``exact`` gives the same outputs in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-6
BLOCK = 16            # tokens that share a scale


# ---- cases -------------------------------------------------------------------------------------


def listed():
    return [
        # one denoised token for each of two players: what counts is the launch
        dict(name="norm_token", op="norm", S=2, Hq=12, Hk=12, D=128, fused=False),
        # a rollout block of ten players (3 frames of 220 tokens each, and the hub tokens)
        dict(name="norm_block", op="norm", S=6678, Hq=24, Hk=24, D=128, fused=False),
        # shared key heads, read in place from one fused projection's rows
        dict(name="norm_shared", op="norm", S=1237, Hq=20, Hk=5, D=64, fused=True),
        # the training step of the four-player clip
        dict(name="norm_grad_clip", op="norm_grad", S=18816, Hq=24, Hk=24, D=128, fused=False),
        # a short clip with shared key heads
        dict(name="norm_grad_shared", op="norm_grad", S=331, Hq=12, Hk=2, D=64, fused=False),
        # the ten-player rollout block into its pages
        dict(name="append_block", op="append", P=10, N=4, L=220, KL=5, KG=6, n=3, W=21, Hk=24, D=128),
        # one frame of two players with few tokens
        dict(name="append_frame", op="append", P=2, N=1, L=37, KL=3, KG=2, n=1, W=7, Hk=6, D=64),
        # the ten-player rollout block with its window full
        dict(name="attend_block", op="attend", P=10, N=4, L=220, KL=5, KG=6, n=3, W=21, Hq=24, Hk=24,
             D=128),
        # four players in two groups
        dict(name="attend_four", op="attend", P=4, N=2, L=220, KL=5, KG=6, n=3, W=21, Hq=12, Hk=12,
             D=128),
        # one player, frame by frame, with a long memory: few rows against many keys
        dict(name="attend_frame", op="attend", P=1, N=1, L=220, KL=5, KG=6, n=1, W=63, Hq=24, Hk=24,
             D=128),
        # a single token against a long cache, with shared key heads
        dict(name="attend_token", op="attend", P=1, N=1, L=1, KL=1, KG=1, n=1, W=4095, Hq=32, Hk=8,
             D=128),
        # odd sizes, shared key heads, a group without members (its hub rows see nothing)
        dict(name="attend_odd", op="attend", P=3, N=2, L=53, KL=3, KG=2, n=2, W=8, Hq=10, Hk=5, D=64),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "append", "attend", "attend"])
    D = rng.choice([64, 128])
    if op in ("norm", "norm_grad"):
        Hk, G = rng.choice([(24, 1), (12, 1), (16, 1), (5, 1), (8, 4), (4, 5), (2, 8), (1, 7)])
        return dict(op=op, S=_spread(rng, 1, 9000), Hq=Hk * G, Hk=Hk, D=D, fused=rng.random() < 0.4)
    n = rng.choice([1, 1, 2, 3])
    if op == "append":
        return dict(op=op, P=rng.randint(1, 8), N=rng.randint(1, 4), L=_spread(rng, 1, 240),
                    KL=rng.randint(1, 7), KG=rng.randint(1, 7), n=n, W=n * rng.randint(1, 6),
                    Hk=rng.choice([1, 3, 8, 12, 24]), D=D)
    Hk, G = rng.choice([(12, 1), (8, 1), (5, 1), (16, 1), (4, 4), (2, 6), (1, 8)])
    P, L = rng.randint(1, 5), _spread(rng, 1, 220)
    # the window in frames so that a player's stream holds up to 8,000 tokens
    frames = _spread(rng, 1, max(1, min(500, 8000 // (n * L))))
    return dict(op=op, P=P, N=rng.randint(1, 3), L=L, KL=rng.randint(1, 6), KG=rng.randint(1, 6), n=n,
                W=n * frames, Hq=Hk * G, Hk=Hk, D=D)


def _labels(c):
    """The group of each player: pairs of neighbours, the last groups left without members."""
    return [min(p // 2, c["N"] - 1) for p in range(c["P"])]


def _active(c):
    lab = _labels(c)
    return [g in lab for g in range(c["N"])]


def _tokens(c):
    return c["P"] * c["n"] * c["L"] + c["n"] * (c["N"] * c["KL"] + c["KG"])


def _frames_seen(c, f):
    """Cached frames that a query of frame f (of the last n of W + n) sees."""
    R = c["W"] + c["n"]
    return R - max(0, f - c["W"] + 1)


def work(case):
    c, D = case, case["D"]
    if case["op"] in ("norm", "norm_grad"):
        vals = c["S"] * (c["Hq"] + c["Hk"]) * D
        table = c["S"] * D * 4                      # cos and sin, D/2 each in fp32
        if c["op"] == "norm":
            return {"bytes": 2 * vals * 2 + table + 2 * D * 4, "flops": 9 * vals}
        return {"bytes": 3 * vals * 2 + table + 4 * D * 4, "flops": 20 * vals}
    S = _tokens(c)
    if c["op"] == "append":
        blocks = c["n"] * (c["P"] * -(-c["L"] // BLOCK) + c["N"] * -(-c["KL"] // BLOCK) + -(-c["KG"] // BLOCK))
        return {"bytes": 2 * c["Hk"] * (S * D * 3 + blocks), "flops": 4 * S * c["Hk"] * D}
    lab, act, R = _labels(c), _active(c), c["W"] + c["n"]
    seen = [_frames_seen(c, R - c["n"] + j) for j in range(c["n"])]
    size = [lab.count(g) for g in range(c["N"])]
    pairs = 0
    for s in seen:
        for p in range(c["P"]):
            pairs += c["L"] * (s * c["L"] + (size[lab[p]] - 1) * c["n"] * c["L"] + s * c["KL"])
        for g in range(c["N"]):
            if act[g]:
                pairs += c["KL"] * s * (size[g] * c["L"] + c["KL"] + c["KG"])
        pairs += c["KG"] * s * (sum(act) * c["KL"] + c["KG"])
    rows = max(seen) * (c["P"] * c["L"] + sum(act) * c["KL"] + c["KG"])
    cached = 2 * c["Hk"] * (rows * D + rows / BLOCK)
    return {"bytes": 2 * S * c["Hq"] * D * 2 + cached, "flops": 4 * c["Hq"] * D * pairs}


# ---- inputs ------------------------------------------------------------------------------------


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _generator(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=_device())


def _norm_inputs(c, seed):
    """Projections, gains near one, angles of the positions, and the gradients of the outputs."""
    g = _generator(seed)
    S, Hq, Hk, D = c["S"], c["Hq"], c["Hk"], c["D"]
    if c["fused"]:
        rows = (_normal(g, S, (Hq + 2 * Hk) * D) * 1.5).to(torch.bfloat16)
        qx, kx = rows[:, :Hq * D], rows[:, Hq * D:(Hq + Hk) * D]
    else:
        qx = (_normal(g, S, Hq * D) * 1.5).to(torch.bfloat16)
        kx = (_normal(g, S, Hk * D) * 0.7).to(torch.bfloat16)
    freq = 10000.0 ** (-torch.arange(D // 2, device=qx.device, dtype=torch.float64) / (D // 2))
    angle = torch.arange(S, device=qx.device, dtype=torch.float64)[:, None] * freq
    st = dict(case=c, qx=qx, kx=kx, wq=1 + 0.2 * _normal(g, D), wk=1 + 0.2 * _normal(g, D),
              cos=torch.cos(angle).float(), sin=torch.sin(angle).float())
    if c["op"] == "norm_grad":
        st["dq"] = (_normal(g, S, Hq, D) * 0.1).to(torch.bfloat16)
        st["dk"] = (_normal(g, S, Hk, D) * 0.1).to(torch.bfloat16)
    return st


def _block_inputs(c, seed, frames):
    """Keys and values of `frames` frames in the cached order [agents | locals by frame | global]:
    channels of unlike size, as norms with gains leave them, and tokens of unlike size."""
    g = _generator(seed)
    S = frames * (c["P"] * c["L"] + c["N"] * c["KL"] + c["KG"])
    H, D = c["Hk"], c["D"]
    make = lambda: (_normal(g, S, H, D) * torch.exp(0.4 * _normal(g, 1, H, D)) *  # noqa: E731
                    torch.exp(0.3 * _normal(g, S, H, 1))).to(torch.bfloat16)
    return g, make(), make()


def _streams(t, c, frames):
    """[P, frames, L, H, D], [N, frames, KL, H, D], [1, frames, KG, H, D] of a block's rows."""
    H, D = t.shape[1:]
    a, l = c["P"] * frames * c["L"], frames * c["N"] * c["KL"]
    return (t[:a].view(c["P"], frames, c["L"], H, D),
            t[a:a + l].view(frames, c["N"], c["KL"], H, D).transpose(0, 1),
            t[a + l:].view(1, frames, c["KG"], H, D))


def _page(width):
    return -(-width // BLOCK) * BLOCK


def _make_cache(c):
    from multics_amd.paged_cache import HierPagedKVCache
    return HierPagedKVCache(num_players=c["P"], num_groups=c["N"], num_patches=c["L"],
                            num_local_hub_tokens=c["KL"], num_global_hub_tokens=c["KG"],
                            num_heads=c["Hk"], head_dim=c["D"], local_attn_size=c["W"],
                            num_frame_per_block=c["n"], device=_device(), dtype=torch.float8_e4m3fn)


def _append_inputs(c, seed):
    """A block's keys and values, and the pages that it goes to: the last of a full ring."""
    _, k, v = _block_inputs(c, seed, c["n"])
    R, n = c["W"] + c["n"], c["n"]
    st = dict(case=c, k=k, v=v, start=2 * R - n, active=[_active(c)] * n)
    if own:
        st["cache"] = _make_cache(c)
        return st
    rows, base, dst = 0, [], []
    for streams, width in ((c["P"], c["L"]), (c["N"], c["KL"]), (1, c["KG"])):
        base.append(rows)
        rows += streams * R * _page(width)
    slot = torch.arange(R - n, R)
    for s, (streams, width) in enumerate(((c["P"], c["L"]), (c["N"], c["KL"]), (1, c["KG"]))):
        page = _page(width)
        dst.append((base[s] + (torch.arange(streams)[:, None, None] * R + slot[:, None]) * page +
                    torch.arange(page)).reshape(-1).to(k.device))
    pool = lambda: torch.zeros(rows, c["Hk"], c["D"], dtype=torch.float8_e4m3fn,  # noqa: E731
                               device=k.device)
    scale = lambda: torch.ones(rows // BLOCK, c["Hk"], device=k.device)  # noqa: E731
    st.update(dst=torch.cat(dst), k_pool=pool(), v_pool=pool(),
              k_scale=scale().to(torch.float8_e8m0fnu), v_scale=scale().to(torch.float8_e8m0fnu))
    return st


def _quantise(x):
    """Codes and scales of [streams, frames, width, H, D] with the width padded to whole blocks:
    [streams, frames, blocks, BLOCK, H, D] e4m3 and [streams, frames, blocks, H].  The scale is the
    smallest power of two (at least 2^-100) that takes the block's largest value to at most 448."""
    s, f, w, H, D = x.shape
    x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, _page(w) - w))
    x = x.reshape(s, f, -1, BLOCK, H, D)
    m, e = torch.frexp(x.abs().amax(dim=(3, 5)))            # amax = m 2^e, m in [1/2, 1)
    e = torch.where(m > 448 / 512, e - 8, e - 9).clamp(min=-100)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    scale = torch.ldexp(torch.ones_like(m), e)
    codes = (x / scale[:, :, :, None, :, None]).to(torch.float8_e4m3fn)
    return codes, scale


def _attend_inputs(c, seed):
    """A cache that W + n frames were appended to, the queries of the last n, and what a program
    keeps for a window: the tile list, or the masks of the plain form."""
    R, n = c["W"] + c["n"], c["n"]
    g, k, v = _block_inputs(c, seed, R)
    q = _normal(g, _tokens(c), c["Hq"], c["D"]).to(torch.bfloat16)
    act = _active(c)
    st = dict(case=c, q=q)
    if own:
        from multics_amd import metadata
        cache = _make_cache(c)
        cache.append(k, v, 0, R, [act] * R)
        st["cache"] = cache
        st["tiles"] = metadata.cached_window_tiles(
            cache, R - 1, device=q.device, n_frames=n, n_block=n, local_attn=c["W"],
            labels=[_labels(c)] * n, q_active=[act] * n, direct_player=True)
        return st
    for name, t in (("k", k), ("v", v)):
        for part, width, x in zip(("agent", "local", "glob"), (c["L"], c["KL"], c["KG"]),
                                  _streams(t, c, R)):
            codes, scale = _quantise(x)
            st[name + "_" + part] = codes.flatten(2, 3)[:, :, :width].contiguous()
            st[name + "_" + part + "_scale"] = scale
    dev = q.device
    lab, act = torch.tensor(_labels(c), device=dev), torch.tensor(act, device=dev)
    qf = torch.arange(R - n, R, device=dev)
    kf = torch.arange(R, device=dev)
    near = (qf[:, None] - kf[None, :]) < c["W"]                                  # [n, R]
    keys = lambda w: near.repeat_interleave(w, dim=1)  # noqa: E731
    tok = torch.arange(c["P"], device=dev)
    mates = (lab[:, None] == lab) & (tok[:, None] != tok)                        # [P, P]
    hub = (lab[:, None] == torch.arange(c["N"], device=dev)) & act               # [P, N]
    P, N, L, KL, KG = c["P"], c["N"], c["L"], c["KL"], c["KG"]
    # players: their own window, their group's tokens of this block, their group's hub
    own_w = keys(L)[None].expand(P, -1, -1)
    block = mates[:, None, :, None].expand(-1, n, -1, n * L).reshape(P, n, -1)
    hubs = (hub[:, None, :, None] & keys(KL)[None, :, None]).reshape(P, n, -1)
    st["agent_mask"] = torch.cat((own_w, block, hubs), 2).repeat_interleave(L, dim=1)
    # a group's hub: its members' windows, its own, the global one
    members = (lab[None] == torch.arange(N, device=dev)[:, None]) & act[:, None]  # [N, P]
    m = (members[:, None, :, None] & keys(L)[None, :, None]).reshape(N, n, -1)
    o = keys(KL)[None] & act[:, None, None]
    w = keys(KG)[None] & act[:, None, None]
    st["local_mask"] = torch.cat((m, o, w), 2).repeat_interleave(KL, dim=1)
    # the global hub: the active groups' hubs, and its own window
    st["glob_mask"] = torch.cat(((act[None, :, None] & keys(KL)[:, None]).reshape(n, -1), keys(KG)),
                                1).repeat_interleave(KG, dim=0)[None]
    return st


def prepare(case, seed):
    make = {"norm": _norm_inputs, "norm_grad": _norm_inputs, "append": _append_inputs,
            "attend": _attend_inputs}
    return make[case["op"]](case, seed)


# ---- the operators -----------------------------------------------------------------------------


def _unit(x, eps=EPS):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _rotate(y, cos, sin):
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _norm(st):
    c = st["case"]
    if own:
        from multics_amd import kernels
        return kernels.qk_head_prologue(
            st["qx"], st["kx"], norm_q_w=st["wq"], norm_k_w=st["wk"], rope_cos=st["cos"],
            rope_sin=st["sin"], num_heads=c["Hq"], num_kv_heads=c["Hk"], eps=EPS)
    cos, sin = st["cos"][:, None], st["sin"][:, None]
    one = lambda x, H, w: _rotate(_unit(x.float().reshape(c["S"], H, -1))[0] * w, cos,  # noqa: E731
                                  sin).to(x.dtype)
    return one(st["qx"], c["Hq"], st["wq"]), one(st["kx"], c["Hk"], st["wk"])


def _norm_grad_one(x, dy, w, cos, sin):
    xf = x.float().reshape(dy.shape)
    xh, r = _unit(xf)
    dn = _rotate(dy.float(), cos, -sin)                     # the rotation's transpose
    dw = (dn * xh).sum((0, 1))
    dh = dn * w
    dx = r * (dh - xh * (dh * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype).reshape(x.shape), dw


def _norm_grad(st):
    c = st["case"]
    if own:
        from multics_amd import kernels
        return kernels.qk_head_prologue_backward(
            st["dq"], st["dk"], st["qx"], st["kx"], norm_q_w=st["wq"], norm_k_w=st["wk"],
            rope_cos=st["cos"], rope_sin=st["sin"], num_heads=c["Hq"], num_kv_heads=c["Hk"], eps=EPS)
    cos, sin = st["cos"][:, None], st["sin"][:, None]
    dqx, dwq = _norm_grad_one(st["qx"], st["dq"], st["wq"], cos, sin)
    dkx, dwk = _norm_grad_one(st["kx"], st["dk"], st["wk"], cos, sin)
    return dqx, dkx, dwq, dwk


def _append(st):
    c = st["case"]
    if own:
        cache = st["cache"]
        cache.append(st["k"], st["v"], st["start"], c["n"], st["active"])
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    # (8-bit tensors are indexed through their bytes)
    byte = lambda t: t.view(torch.uint8)  # noqa: E731
    at = st["dst"][::BLOCK] // BLOCK
    for name in ("k", "v"):
        parts = [_quantise(x) for x in _streams(st[name], c, c["n"])]
        codes = torch.cat([byte(q).flatten(0, 3) for q, _ in parts])
        scale = torch.cat([s.flatten(0, 2) for _, s in parts]).to(torch.float8_e8m0fnu)
        byte(st[name + "_pool"])[st["dst"]] = codes
        byte(st[name + "_scale"])[at] = byte(scale)
    return st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"]


def _held(st, name, part):
    """[streams, tokens, H, D] fp32: the values that the codes of a kind of stream stand for."""
    codes, scale = st[name + "_" + part], st[name + "_" + part + "_scale"]
    each = scale.repeat_interleave(BLOCK, dim=2)[:, :, :codes.shape[2]]
    return (codes.float() * each[..., None]).flatten(1, 2)


def _softmax_rows(q, k, v, mask):
    """q [B, n, Hq, D], k / v [B, m, Hk, D], mask [B, n, m]: rows that see nothing give zero."""
    G = q.shape[2] // k.shape[2]
    heads = lambda t, r: t.repeat_interleave(r, dim=2).transpose(1, 2)  # noqa: E731
    s = torch.matmul(heads(q.float(), 1), heads(k, G).transpose(2, 3).contiguous())
    s = (s / math.sqrt(q.shape[-1])).masked_fill_(~mask[:, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, heads(v, G).contiguous())
    return (o / torch.where(total > 0, total, torch.ones_like(total))).transpose(1, 2).to(q.dtype)


def _attend(st):
    c, q = st["case"], st["q"]
    if own:
        from multics_amd import kernels
        return kernels.hier_cached_attention_fp8(q, st["cache"], st["tiles"])
    P, N, n, L = c["P"], c["N"], c["n"], c["L"]
    agent, local, glob = ((_held(st, "k", part), _held(st, "v", part))
                          for part in ("agent", "local", "glob"))
    # one row of streams for all: every stream that reads another's keys reads them whole
    row = lambda t, times: t.flatten(0, 1)[None].expand(times, -1, -1, -1)  # noqa: E731
    qa, ql, qg = _streams(q, c, n)
    one = lambda t: t.flatten(1, 2)  # noqa: E731
    a = _softmax_rows(one(qa), *(torch.cat((x, row(x[:, -n * L:], P), row(y, P)), 1)
                                 for x, y in zip(agent, local)), st["agent_mask"])
    b = _softmax_rows(one(ql), *(torch.cat((row(x, N), y, z.expand(N, -1, -1, -1)), 1)
                                 for x, y, z in zip(agent, local, glob)), st["local_mask"])
    d = _softmax_rows(one(qg), *(torch.cat((row(y, 1), z), 1) for y, z in zip(local, glob)),
                      st["glob_mask"])
    b = b.view(N, n, c["KL"], *q.shape[1:]).transpose(0, 1)
    return torch.cat((a.flatten(0, 1), b.flatten(0, 2), d.flatten(0, 1)))


def run(state):
    return {"norm": _norm, "norm_grad": _norm_grad, "append": _append,
            "attend": _attend}[state["case"]["op"]](state)


# ---- the same in 64 bits -----------------------------------------------------------------------


def _exact_norm(c, seed):
    """The rotation as a product of complex numbers; gradients by differentiating it."""
    st = _norm_inputs(c, seed)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[:, None]
    wide = [st[k].double().contiguous().requires_grad_(c["op"] == "norm_grad")
            for k in ("qx", "kx", "wq", "wk")]
    outs = []
    for x, w, H in ((wide[0], wide[2], c["Hq"]), (wide[1], wide[3], c["Hk"])):
        h = x.view(c["S"], H, c["D"])
        y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / c["D"] + EPS) * w
        z = torch.view_as_complex(y.view(c["S"], H, c["D"] // 2, 2)) * turn
        outs.append(torch.view_as_real(z).flatten(-2))
    if c["op"] == "norm":
        return tuple(outs)
    return torch.autograd.grad(outs, wide, [st["dq"].double(), st["dk"].double()])


def _exact_codes(x):
    """Codes and scale of one block [tokens, H, D]: the exponent by trying, the code as a multiple of
    its step, all in 64 bits."""
    x = x.double()
    top = x.abs().amax(dim=(0, 2))
    e = torch.full_like(top, -100.0)
    for up in (128, 64, 32, 16, 8, 4, 2, 1):                # the largest e - 1 that is too small
        e = torch.where(top > 448 * torch.exp2(e + up - 1), e + up, e)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    scale = torch.exp2(e)
    y = x / scale[:, None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale


def _exact_append(c, seed):
    _, k, v = _block_inputs(c, seed, c["n"])
    R, n, out = c["W"] + c["n"], c["n"], []
    widths = ((c["P"], c["L"]), (c["N"], c["KL"]), (1, c["KG"]))
    rows = sum(s * R * _page(w) for s, w in widths)
    for t in (k, v):
        pool = torch.zeros(rows, c["Hk"], c["D"], dtype=torch.float64, device=t.device)
        scale = torch.ones(rows // BLOCK, c["Hk"], dtype=torch.float64, device=t.device)
        base = 0
        for (streams, w), x in zip(widths, _streams(t, c, n)):
            for s in range(streams):
                for j in range(n):
                    at = base + (s * R + R - n + j) * _page(w)
                    for b in range(0, w, BLOCK):
                        codes, sc = _exact_codes(x[s, j, b:b + BLOCK])
                        pool[at + b:at + b + codes.shape[0]] = codes
                        scale[(at + b) // BLOCK] = sc
            base += streams * R * _page(w)
        out.append((pool, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_values(t, c, R):
    """What the cache holds of each stream's tokens, [streams][frames * width, H, D]."""
    kinds = []
    for x in _streams(t, c, R):
        s, f, w, H, D = x.shape
        held = torch.empty(s, f, w, H, D, dtype=torch.float64, device=x.device)
        for b in range(0, w, BLOCK):                        # all pages at once: [tokens, pages * H, D]
            part = x[:, :, b:b + BLOCK].permute(2, 0, 1, 3, 4)
            codes, scale = _exact_codes(part.reshape(part.shape[0], -1, D))
            held[:, :, b:b + BLOCK] = (codes * scale[:, None]).view(part.shape).permute(1, 2, 0, 3, 4)
        kinds.append(held.flatten(1, 2))
    return kinds


def _exact_attend(c, seed):
    """Stream by stream: the keys that its rows may see are gathered, frames compared one by one."""
    R, n, D = c["W"] + c["n"], c["n"], c["D"]
    g, k, v = _block_inputs(c, seed, R)
    q = _normal(g, _tokens(c), c["Hq"], D).to(torch.bfloat16).double()
    K, V = _exact_values(k, c, R), _exact_values(v, c, R)
    lab, act = _labels(c), _active(c)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    width = (c["L"], c["KL"], c["KG"])

    def answer(rows, frame, parts):
        """parts: (kind, stream, first frame) of the keys that may be seen within the window."""
        frames = [f for f in range(R) if frame - f < c["W"]]
        idx = []
        for kind, s, since in parts:
            w = width[kind]
            first = max([since] + frames[:1])
            idx.append((K[kind][s][first * w:], V[kind][s][first * w:]))
        if not idx:
            return
        kk, vv = (torch.cat([x[i] for x in idx]) for i in (0, 1))
        G = c["Hq"] // c["Hk"]
        for h in range(c["Hk"]):
            qq = q[rows][:, h * G:(h + 1) * G]
            s = torch.einsum("rgd,kd->rgk", qq, kk[:, h]) * D ** -0.5
            out[rows, h * G:(h + 1) * G] = torch.einsum("rgk,kd->rgd", torch.softmax(s, -1), vv[:, h])

    row = lambda a, w: torch.arange(a, a + w, device=q.device)  # noqa: E731
    a_end, l_end = c["P"] * n * c["L"], c["P"] * n * c["L"] + n * c["N"] * c["KL"]
    for j in range(n):
        f = R - n + j
        for p in range(c["P"]):
            parts = [(0, p, 0)] + [(0, o, R - n) for o in range(c["P"]) if o != p and lab[o] == lab[p]]
            answer(row((p * n + j) * c["L"], c["L"]), f, parts + [(1, lab[p], 0)])
        for gr in range(c["N"]):
            if act[gr]:
                parts = [(0, p, 0) for p in range(c["P"]) if lab[p] == gr]
                answer(row(a_end + (j * c["N"] + gr) * c["KL"], c["KL"]), f,
                       parts + [(1, gr, 0), (2, 0, 0)])
        answer(row(l_end + j * c["KG"], c["KG"]), f,
               [(1, gr, 0) for gr in range(c["N"]) if act[gr]] + [(2, 0, 0)])
    return out


def exact(case, seed):
    return {"norm": _exact_norm, "norm_grad": _exact_norm, "append": _exact_append,
            "attend": _exact_attend}[case["op"]](case, seed)
