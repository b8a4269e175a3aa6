"""The KV cache held in 8 bits on the GPU: the append against its definition
(every code and scale), the attention against a softmax in 64 bits over the
values that the cache stands for, and both with the per-head norms in a rollout.

Bounds of the attention, per element, with weights w (their sum 1): a weight is
rounded to bf16 (at most 2^-8 of it) and the row sum adds the rounded weights,
so the result moves by at most 2^-8 of sum w |v - o|; the result is rounded to
bf16 (2^-8 of it); the scores are fp32 sums (fewer than 2^8 roundings of 2^-24
of |q| |k|, and the two codes of q leave at most 2^-22 of its largest element),
which for the sizes here (|q| |k| / sqrt(D) below 2^6) is less than 2^-9 in a
score only for keys whose weight vanishes, and 2^-13 on average: 2^-11 of
sum w |v|.  The normaliser adds rounded weights: 2^-8 (relative), 2^-8 in lse.
"""

import numpy as np
import pytest
import torch

from multics_amd import kernels
from multics_amd import metadata as M
from multics_amd.kernels import (hier_attention_forward, hier_cached_attention_fp8,
                                 qk_head_prologue)
from multics_amd.module import SelfAttention
from multics_amd.paged_cache import HierPagedKVCache
from tests.gpu_util import expand_tiles, need_gpu, say

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
STEP = 2.0 ** -8


def _cache(P=2, N=2, L=37, KL=3, KG=5, H=3, D=64, W=4, n=2, dtype=FP8, **kw):
    return HierPagedKVCache(num_players=P, num_groups=N, num_patches=L, num_local_hub_tokens=KL,
                            num_global_hub_tokens=KG, num_heads=H, head_dim=D, local_attn_size=W,
                            num_frame_per_block=n, device="cuda", dtype=dtype, **kw)


def _rows(c, n):
    return c.P * n * c.L + n * (c.N * c.KL + c.KG)


def _define(x, bad):
    """Codes and exponents of blocks [blocks, 16, D] from the definition, in 64
    bits; ``bad`` [blocks, 16]: tokens kept as not a number (counted as 0)."""
    x = np.where(bad[:, :, None], 0.0, x.astype(np.float64))
    top = np.abs(x).max((1, 2))
    e = np.full(top.shape, -100)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):
        e = np.where(top > 448 * np.exp2(e + step - 1.0), e + step, e)
    e = np.where(top == 0, 0, e)
    y = x / np.exp2(e.astype(np.float64))[:, None, None]
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.rint(y / step) * step, e


def _special(k, v, seed):
    """Values that a rounding or a scale can go wrong at, over random ones."""
    rng = np.random.default_rng(seed)
    k, v = k.clone(), v.clone()
    S, H, D = k.shape
    k[0, 0] = 0
    k[:16, H - 1] = 0                                       # a block of zeros
    v[3, 0, :4] = torch.tensor([448.0, -448.0, 2.0 ** -9, 2.0 ** -10], dtype=torch.bfloat16)
    k[5, 0, 0] = 3.0e38
    v[6, 0, 1] = 1e-38
    k[8, 0, 2] = 2.0 ** -133                                # the smallest bf16
    ties = torch.tensor([1.0625, 1.1875, 17.0, 19.0, -1.0625, 208.0, 216.0, 232.0],
                        dtype=torch.bfloat16)               # halves of e4m3's steps
    v[9, :, 8:16] = ties
    v[10, :, 8:16] = ties * 2.0 ** -13
    return k, v, rng


@pytest.mark.parametrize("D,H,L", [(64, 3, 37), (128, 5, 16), (128, 1, 1), (64, 9, 47)])
def test_append_is_the_definition(D, H, L):
    need_gpu()
    c = _cache(L=L, H=H, D=D)
    n, S = 2, _rows(_cache(L=L, H=H, D=D), 2)
    g = torch.Generator(device="cuda").manual_seed(D + L)
    mk = lambda: (torch.randn(S, H, D, generator=g, device="cuda") *  # noqa: E731
                  torch.exp(3 * torch.randn(S, H, 1, generator=g, device="cuda"))).to(torch.bfloat16)
    k, v = mk(), mk()
    if S > 16:
        k, v, rng = _special(k, v, L)
        k[S - 2, 0, 5] = float("nan")
        v[S - 4, H - 1, D - 1] = float("-inf")
        v[20 % S, 0, 0] = float("nan")
    say("fp8 append", D, H, L)
    held = c.k.view(torch.uint8).clone(), c.k_scale.view(torch.uint8).clone()
    c.append(k, v, 5, n, np.ones((n, 2), bool))
    torch.cuda.synchronize()
    table = c.block_table(5, n)
    pad = lambda t: np.stack([np.pad(t[s:s + m], ((0, 16 - m), (0, 0), (0, 0)))  # noqa: E731
                              for s, _, m in table])        # [blocks, 16, H, D]
    kb, vb = (pad(t.float().cpu().numpy()) for t in (k, v))
    bad = ~(np.isfinite(kb).all(-1) & np.isfinite(vb).all(-1))           # [blocks, 16, H]
    for name, x, pool, scale in (("k", kb, c.k, c.k_scale), ("v", vb, c.v, c.v_scale)):
        pool, scale = pool.double().cpu().numpy(), scale.double().cpu().numpy()
        for h in range(H):
            codes, e = _define(np.nan_to_num(x[:, :, h]), bad[:, :, h])
            if name == "k":
                codes[bad[:, :, h]] = np.nan
            for b, (_, d, m) in enumerate(table):
                assert scale[d // 16, h] == 2.0 ** e[b], (name, h, b)
                assert np.array_equal(pool[d:d + m, h], codes[b, :m], equal_nan=True), (name, h, b)
    # what no block row reaches is as it was: other pages, and rows behind a page's tokens
    rows = torch.from_numpy(c.block_rows(5, n)).long().cuda()
    other = torch.ones(c.k.shape[0], dtype=torch.bool, device="cuda")
    other[rows] = False
    assert torch.equal(c.k.view(torch.uint8)[other], held[0][other])
    blocks = torch.ones(c.k_scale.shape[0], dtype=torch.bool, device="cuda")
    blocks[torch.from_numpy(table[:, 1] // 16).long().cuda()] = False
    assert torch.equal(c.k_scale.view(torch.uint8)[blocks], held[1][blocks])


def test_append_reads_views_and_repeats_itself():
    need_gpu()
    S = _rows(_cache(), 2)
    g = torch.Generator(device="cuda").manual_seed(1)
    whole = torch.randn(3, 2, S, 64, generator=g, device="cuda").to(torch.bfloat16)
    k, v = whole[:, 0].transpose(0, 1), whole[:, 1].transpose(0, 1)     # head-major slices
    odd = torch.randn(S, 3, 65, generator=g, device="cuda").to(torch.bfloat16)[:, :, 1:]
    act = np.ones((2, 2), bool)
    for a, b in ((k, v), (odd, k)):
        one, two = _cache(), _cache()
        one.append(a, b, 0, 2, act)
        two.append(a.contiguous(), b.contiguous(), 0, 2, act)
        two.append(a.contiguous(), b.contiguous(), 0, 2, act)           # a re-run: the same pages
        for x, y in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # values of an 8-bit cache go in and out unchanged
    kd, vd = one.dequantised()
    rows = torch.from_numpy(one.block_rows(0, 2)).long().cuda()
    two.append(kd[rows], vd[rows], 0, 2, act)
    assert torch.equal(two.dequantised()[0], kd) and torch.equal(two.dequantised()[1], vd)


# ---- attention ------------------------------------------------------------------------------

CASES = [
    # name, P, N, L, KL, KG, n, W, Hk, G, D, frames, labels, active
    ("block", 3, 2, 53, 3, 2, 2, 6, 3, 1, 128, 8, [0, 0, 1], [True, True]),
    ("d64_shared", 3, 2, 53, 3, 2, 2, 6, 2, 3, 64, 10, [0, 0, 1], [True, True]),
    ("token", 1, 1, 1, 1, 1, 1, 300, 2, 4, 128, 301, [0], [True]),
    ("first_token", 1, 1, 1, 1, 1, 1, 4, 1, 1, 64, 1, [0], [True]),
    ("empty_group", 2, 2, 40, 4, 3, 3, 3, 2, 1, 64, 6, [0, 0], [True, False]),
    ("long", 2, 1, 130, 5, 6, 1, 40, 1, 1, 128, 41, [0, 0], [True]),
    ("wrapped", 2, 1, 33, 2, 1, 2, 4, 2, 2, 128, 16, [0, 0], [True]),
]


def _rollout(case, seed=0, hide=None, batch=1, dtype=FP8):
    """A cache with ``frames`` appended block by block, the last block's list."""
    _, P, N, L, KL, KG, n, W, Hk, G, D, frames, labels, active = case
    c = _cache(P, N, L, KL, KG, Hk, D, W, n, dtype=dtype, batch=batch)
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, HB = _rows(c, n), Hk * batch
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    act = [active] * n
    for f in range(0, frames, n):
        k = (rnd(S, HB, D) * torch.exp(0.5 * rnd(1, HB, D))).to(torch.bfloat16)
        v = (rnd(S, HB, D) * torch.exp(0.5 * rnd(S, HB, 1)) + 0.3).to(torch.bfloat16)
        if hide is not None:
            hide(c, f, k, v)
        c.append(k, v, f, n, act)
    q = rnd(S, HB * G, D).to(torch.bfloat16)
    tiles = M.cached_window_tiles(c, frames - 1, device="cuda", n_frames=n, n_block=n, local_attn=W,
                                  labels=[labels] * n, q_active=act, direct_player=True)
    return c, q, tiles


def _reference(q, c, tiles, scale=None):
    """(o, bound, lse) [S, H, D] / [H, S] of a softmax in 64 bits over the keys that
    each row sees by the list."""
    k, v = (t.double().transpose(0, 1) for t in c.dequantised())
    S, H, D = q.shape
    seen = torch.zeros(S, k.shape[1], dtype=torch.bool)
    for r, keys in expand_tiles(tiles).items():
        seen[r, sorted(keys)] = True
    seen = seen.cuda()
    G = H // k.shape[0]
    scale = D ** -0.5 if scale is None else scale
    o, bound = torch.zeros(S, H, D, dtype=torch.float64).cuda(), None
    bound, lse = torch.zeros_like(o), torch.full((H, S), float("-inf"), dtype=torch.float64).cuda()
    some = seen.any(1)
    for h in range(H):
        kk, vv = k[h // G], v[h // G]
        s = (q[:, h].double() @ kk.t().contiguous()) * scale
        s = torch.where(seen, s, torch.full_like(s, float("-inf")))[some]
        w = torch.softmax(s, -1)
        # keys that nobody in a row sees have w = 0 and count for nothing
        w = torch.where(seen[some], w, torch.zeros_like(w))
        vv = torch.where(seen.any(0)[:, None], vv, torch.zeros_like(vv))
        o[some, h] = w @ vv
        dev = torch.stack([(w[i][:, None] * (vv - o[some, h][i]).abs()).sum(0)
                           for i in range(w.shape[0])])
        bound[some, h] = STEP * (dev + o[some, h].abs()) + 2.0 ** -11 * (w @ vv.abs())
        lse[h, some] = torch.logsumexp(s, -1)
    return o, bound, lse


def _check(q, c, tiles, scale=None):
    S, H, _ = q.shape
    lse = torch.full((H, S), 7.0, device="cuda")
    out = hier_cached_attention_fp8(q, c, tiles, lse=lse, scale=scale)
    torch.cuda.synchronize()
    ref, bound, rlse = _reference(q, c, tiles, scale)
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-30)).max())
    empty = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse), empty)
    assert bool(((lse.double() - rlse)[~empty].abs() <= STEP + 2.0 ** -11).all())
    return out, lse


@pytest.mark.parametrize("splits", [1, 3, 32, None])
@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_attention_matches_64_bits(case, splits, monkeypatch):
    need_gpu()
    if splits is not None:
        monkeypatch.setattr(kernels, "_fp8_splits", lambda workgroups, max_tiles: splits)
    c, q, tiles = _rollout(case)
    say("fp8 attention", case[0], splits)
    out, lse = _check(q, c, tiles)
    again = hier_cached_attention_fp8(q, c, tiles)
    assert torch.equal(out, again)
    if case[0] == "empty_group":
        n, P, L, KL = case[6], case[1], case[3], case[4]
        hub = out[P * n * L:P * n * L + n * 2 * KL].view(n, 2, KL, -1)
        assert torch.count_nonzero(hub[:, 1]) == 0 and torch.count_nonzero(hub[:, 0]) > 0
    # near the bf16 kernel over the same values: each within its bound
    k, v = (t.contiguous() for t in c.dequantised())
    if q.shape[1] == k.shape[1]:
        wide = torch.zeros_like(out)
        hier_attention_forward(q, k, v, tiles, wide)
        _, bound, _ = _reference(q, c, tiles)
        assert bool(((wide.double() - out.double()).abs() <= 2 * bound).all())


def test_membership_batch_and_scale():
    """Two prompts' caches in one pool, a membership topology, another scale."""
    need_gpu()
    P, N, L, KL, KG, n, W, H, D = 3, 2, 21, 2, 3, 2, 4, 2, 64
    mem = np.zeros((4, N, P), bool)
    mem[:, 0, 0] = mem[:, 0, 1] = mem[:, 1, 1] = True
    go = ~mem.any(1)
    c = _cache(P, N, L, KL, KG, H, D, W, n, batch=2)
    g = torch.Generator(device="cuda").manual_seed(5)
    S = _rows(c, n)
    mk = lambda: torch.randn(S, 2 * H, D, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    for f in (0, 2):
        c.append(mk(), mk(), f, n, mem.any(-1)[f:f + n])
    tiles = M.cached_window_tiles(c, 3, device="cuda", n_frames=n, n_block=n, local_attn=W,
                                  labels=None, q_active=mem.any(-1)[2:4], direct_player=True,
                                  membership=mem, global_only=go)
    _check(mk(), c, tiles, scale=0.3)


@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_queries_of_any_size(size):
    """The two codes of a query scale with its row; large scores pick one key."""
    need_gpu()
    c, q, tiles = _rollout(CASES[0], seed=3)
    q = (q.double() * size).to(torch.bfloat16)
    q[:, :, 0] = 0
    q[5] = 0
    _check(q, c, tiles, scale=1 / size / 128 ** 0.5)


def test_hidden_keys_add_nothing_whatever_they_hold():
    need_gpu()
    case = CASES[0]                # players 0, 1 in group 0, player 2 in group 1
    L, n = case[3], case[6]
    mine = 2 * n * L + 17          # a token of player 2

    def hide(value):
        def put(c, f, k, v):
            k[mine], v[mine] = value, value
            k[mine + 1, 1, 3] = v[mine + 2, 1, 5] = value
        return put

    outs = []
    for value in (0.0, float("nan"), float("inf"), float("-inf")):
        c, q, tiles = _rollout(case, hide=hide(value))
        outs.append(hier_cached_attention_fp8(q, c, tiles))
    seen = expand_tiles(tiles)
    bad = [int(r) for f in range(c.R) for r in c.block_rows(f, 1)[2 * L:3 * L][17:20]]
    sees = torch.tensor([bool(seen.get(r, set()) & set(bad)) for r in range(q.shape[0])])
    assert sees.any() and not sees.all()
    for out in outs[1:]:
        # (in head 1 the marks in one channel count as zeros for the scales: other
        # keys of their blocks may be held on another scale than with a zero there)
        assert torch.equal(out[~sees][:, 0], outs[0][~sees][:, 0])
        assert bool(torch.isfinite(out[~sees]).all()) and bool(torch.isnan(out[sees][:, 0]).all())
    assert all(torch.equal(a.view(torch.int16), outs[1].view(torch.int16)) or
               torch.equal(torch.isnan(a), torch.isnan(outs[1])) for a in outs[1:])


def test_queries_that_are_not_numbers_stay_in_their_row():
    """A query with a NaN or an infinity gives NaN, and every other row and head
    what it gave without it (a list of long items and one of few rows)."""
    need_gpu()
    for case in (CASES[0], CASES[1], CASES[2]):
        c, q, tiles = _rollout(case)
        want = hier_cached_attention_fp8(q, c, tiles)
        bad = torch.zeros(want.shape[:2], dtype=torch.bool, device="cuda")
        for i, value in enumerate((float("nan"), float("inf"), float("-inf"))):
            row, head = (7 * i) % q.shape[0], i % q.shape[1]
            q[row, head, 3 + i] = value
            bad[row, head] = True
        got = hier_cached_attention_fp8(q, c, tiles)
        assert bool(torch.isnan(got[bad]).all()), case[0]
        assert torch.equal(got[~bad], want[~bad]), case[0]


def test_two_calls_at_once_on_two_streams():
    """One cache and one new list read from two streams at a time: each call has
    its own workspace, and the list made on one stream is waited for on the other."""
    need_gpu()
    c, q, tiles = _rollout(CASES[5])           # key lists in parts
    qs = [q, (q.float() * 1.5).to(torch.bfloat16)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(hier_cached_attention_fp8(qs[i], c, tiles))
    torch.cuda.synchronize()
    for i in range(2):
        want = hier_cached_attention_fp8(qs[i], c, tiles)
        assert all(torch.equal(o, want) for o in outs[i])
    _check(qs[1], c, tiles)


def test_in_and_out_of_inference_mode():
    """A cache, its list and the list's launch order made in inference mode serve
    calls outside of it, and the other way round."""
    need_gpu()
    case, outs = CASES[0], []
    for made, called in ((True, False), (False, True), (False, False)):
        M.clear_metadata_cache()
        with torch.inference_mode(made):
            c, q, tiles = _rollout(case)
            outs.append(hier_cached_attention_fp8(q, c, tiles))
        with torch.inference_mode(called), torch.no_grad():
            c.append(q, q, case[11] - case[6], case[6], [case[13]] * case[6])
            outs.append(hier_cached_attention_fp8(q, c, tiles))
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[0], outs[4])
    assert torch.equal(outs[1], outs[3]) and torch.equal(outs[1], outs[5])
    assert not torch.equal(outs[0], outs[1])


def test_a_pool_past_32_bits():
    """Pools of more than 2^32 bytes, the rows in use at their far end: codes,
    scales and outputs as in a small cache that holds the same frames."""
    need_gpu()
    kw = dict(P=1, N=1, L=1000, KL=1, KG=1, H=32, D=128, n=1)
    small, big = _cache(W=2, **kw), _cache(W=1100, **kw)
    assert big.k.shape[0] * 32 * 128 > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(11)
    S = _rows(big, 1)
    mk = lambda: torch.randn(S, 32, 128, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    for f in range(big.R - 3, big.R):          # the last pages of the ring
        k, v = mk(), mk()
        big.append(k, v, f, 1, [[True]])
        small.append(k, v, f, 1, [[True]])
    q, outs = mk(), []
    for c in (small, big):
        tiles = M.cached_window_tiles(c, big.R - 1, device="cuda", n_frames=1, n_block=1, local_attn=2,
                                      labels=[[0]], q_active=[[True]], direct_player=True)
        outs.append(hier_cached_attention_fp8(q, c, tiles))
        rows = [torch.from_numpy(c.block_rows(f, 1)).long().cuda() for f in range(big.R - 3, big.R)]
        outs.append([(t.view(torch.uint8)[r].clone(), s.view(torch.uint8)[r // 16].clone())
                     for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)) for r in rows])
    assert torch.equal(outs[0], outs[2]) and torch.count_nonzero(outs[0]) > 0
    assert all(torch.equal(a, b) for x, y in zip(outs[1], outs[3]) for a, b in zip(x, y))


def test_rows_of_no_item_and_views():
    need_gpu()
    c, q, tiles = _rollout(CASES[0])
    S, H, D = q.shape
    out = hier_cached_attention_fp8(q, c, tiles)
    room = torch.full((S + 9, H, D), 3.0, dtype=torch.bfloat16, device="cuda")
    big = torch.zeros(H, S + 9, D + 8, dtype=torch.bfloat16, device="cuda").transpose(0, 1)[:, :, :D]
    big[:S] = q
    got = hier_cached_attention_fp8(big, c, tiles, out=room)
    assert got is room and torch.equal(room[:S], out) and bool((room[S:] == 3).all())
    assert torch.count_nonzero(hier_cached_attention_fp8(big, c, tiles)[S:]) == 0
    odd = torch.zeros(S, H, D + 3, dtype=torch.bfloat16, device="cuda")[:, :, 3:]
    odd.copy_(q)
    assert torch.equal(hier_cached_attention_fp8(odd, c, tiles), out)
    four = hier_cached_attention_fp8(q[None], c, tiles, out=torch.empty_like(q)[None])
    assert torch.equal(four[0], out)


def test_one_token_of_one_head_with_strides_of_no_meaning():
    """A dimension of one element may have any stride."""
    need_gpu()
    case = CASES[3]
    c, q, tiles = _rollout(case)
    S, H, D = q.shape
    assert H == 1
    want = hier_cached_attention_fp8(q, c, tiles)
    odd = q.as_strided((S, 1, D), (D, 1, 1))
    got = hier_cached_attention_fp8(odd, c, tiles, out=torch.zeros_like(q).as_strided((S, 1, D), (D, 3, 1)))
    assert torch.equal(got, want)
    one, two = _cache(1, 1, 1, 1, 1, 1, 64, 4, 1), _cache(1, 1, 1, 1, 1, 1, 64, 4, 1)
    k = torch.randn(3, 1, 64, device="cuda").to(torch.bfloat16)
    one.append(k, k, 0, 1, [[True]])
    two.append(k.as_strided((3, 1, 64), (64, 5, 1)), k, 0, 1, [[True]])
    assert torch.equal(one.k.view(torch.uint8), two.k.view(torch.uint8))


def test_refusals():
    need_gpu()
    c, q, tiles = _rollout(CASES[0])
    S, H, D = q.shape
    for exc, args, kw in [
        (ValueError, (q[:, :2], c, tiles), {}), (ValueError, (q[:, :, :64], c, tiles), {}),
        (ValueError, (q[:-1], c, tiles), {}), (ValueError, (q, c, tiles), {"out": q[:-1].clone()}),
        (ValueError, (q, c, tiles), {"out": q.float()}),
        (ValueError, (q, c, tiles), {"out": torch.empty(S, D, H, device="cuda",
                                                        dtype=torch.bfloat16).transpose(1, 2)}),
        (ValueError, (q, c, tiles), {"lse": torch.empty(H, S - 1, device="cuda")}),
        (ValueError, (q, c, tiles), {"lse": torch.empty(H, S)}),
        (ValueError, (q, c, tiles), {"scale": 0.0}), (ValueError, (q, c, tiles), {"scale": -1.0}),
        (ValueError, (q, c, tiles), {"scale": float("nan")}), (ValueError, (q[0], c, tiles), {}),
        (NotImplementedError, (q.half(), c, tiles), {}),
        (ValueError, (q, _cache(2, 1, 33, 2, 1, 3, 128, 2, 2), tiles), {}),
    ]:
        with pytest.raises(exc):
            hier_cached_attention_fp8(*args, **kw)


def test_norm_append_attend_together_in_a_graph():
    """The three of a block captured once on a side stream and replayed on new
    projections, with eager calls between the replays: equal bits."""
    need_gpu()
    case = CASES[1]
    _, P, N, L, KL, KG, n, W, Hk, G, D, frames, labels, active = case
    c, _, tiles = _rollout(case)
    S = _rows(c, n)
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = (1 + 0.1 * rnd(D)).to(torch.bfloat16)
    angle = rnd(S, D // 2)
    kw = dict(norm_q_w=w, norm_k_w=w, rope_cos=angle.cos(), rope_sin=angle.sin(), eps=1e-6,
              num_heads=Hk * G, num_kv_heads=Hk)
    fused = rnd(S, (Hk * G + 2 * Hk) * D).to(torch.bfloat16)
    cols = lambda a, b: fused[:, a * D:b * D]  # noqa: E731

    def block():
        q, k = qk_head_prologue(cols(0, Hk * G), cols(Hk * G, Hk * G + Hk), **kw)
        v = cols(Hk * G + Hk, Hk * G + 2 * Hk).reshape(S, Hk, D)
        c.append(k, v, frames - n, n, [active] * n)
        return hier_cached_attention_fp8(q, c, tiles)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for _ in range(4):
        fused.copy_(rnd(*fused.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, block())
        say("replayed")


@pytest.mark.parametrize("qk_norm", ["head", "model"])
def test_module_rollout_over_an_8_bit_cache(qk_norm, monkeypatch):
    """``SelfAttention.causal_forward`` with such a cache is its parts: norms,
    append, attention, o-projection; blocks in turn and one re-run; both
    prompts in one cache of batch 2 (equal bits when the key lists are cut
    alike: how many parts they are cut into goes by the number of heads, and a
    part's weights are rounded against its own running max)."""
    need_gpu()
    monkeypatch.setattr(kernels, "_fp8_splits", lambda workgroups, max_tiles: 2)
    P, N, L, KL, KG, n, W, H, D = 3, 2, 21, 2, 3, 2, 4, 4, 64
    torch.manual_seed(0)
    m = SelfAttention(H * D, H, qk_norm=qk_norm).to("cuda", torch.bfloat16).eval()
    m.num_frame_per_block, m.local_attn_size = n, W
    # the o-projection leaves its input: a GEMM sums another way for two prompts
    # than for one
    torch.nn.init.eye_(m.o.weight)
    torch.nn.init.zeros_(m.o.bias)
    caches = [_cache(P, N, L, KL, KG, H, D, W, n) for _ in range(2)]
    pair = _cache(P, N, L, KL, KG, H, D, W, n, batch=2)
    S = _rows(caches[0], n)
    labels = torch.tensor([[0, 0, 1]] * n)
    with torch.no_grad():
        for f in (0, 2, 4, 6, 6):
            x = torch.randn(2, S, H * D, device="cuda").to(torch.bfloat16)
            freqs = torch.polar(torch.ones(S, 1, D // 2, dtype=torch.float64, device="cuda"),
                                torch.rand(S, 1, D // 2, dtype=torch.float64, device="cuda"))
            kw = dict(current_start=f * P * L, num_frames=n, num_players=P, group_labels=labels,
                      direct_player=True)
            ys = [m.causal_forward(x[i:i + 1], freqs, kv_cache=caches[i], **kw) for i in range(2)]
            both = m.causal_forward(x, freqs, kv_cache=pair, **kw)
            q, k, v = m._qkv_blocks(x[:1], freqs, None)
            c = _cache(P, N, L, KL, KG, H, D, W, n)
            for name in ("k", "v", "k_scale", "v_scale"):
                getattr(c, name).view(torch.uint8).copy_(getattr(caches[0], name).view(torch.uint8))
            rows = torch.from_numpy(c.block_rows(f, n)).long().cuda()
            c.k.view(torch.uint8)[rows] = 0
            c.slot_frame[:], c.local_active[:] = caches[0].slot_frame, caches[0].local_active
            c.append(k, v, f, n, [[True, True]] * n)
            tiles = M.cached_window_tiles(c, f + n - 1, device="cuda", n_frames=n, n_block=n,
                                          local_attn=W, labels=labels.numpy(),
                                          q_active=np.ones((n, N), bool), direct_player=True)
            y, _ = _check(q, c, tiles)
            assert torch.equal(m.o(y.reshape(1, S, -1)), ys[0])
            assert torch.equal(torch.cat(ys), both)
            for i in range(2):
                assert torch.equal(pair.k[:, i * H:(i + 1) * H].float(), caches[i].k.float())


def test_an_index_list_may_start_anywhere():
    """Pool rows are read one at a time: a list of them that starts at any entry of
    an array serves; a mask list that cannot be read 16 bytes at a time is refused."""
    need_gpu()
    import dataclasses
    shifted = lambda t: torch.cat((t[:1], t))[1:]  # noqa: E731
    for case in (CASES[0], CASES[2]):
        c, q, tiles = _rollout(case)
        want = hier_cached_attention_fp8(q, c, tiles)
        odd = dataclasses.replace(tiles, kv_idx=shifted(tiles.kv_idx))
        assert odd.kv_idx.data_ptr() % 16 == 4
        assert torch.equal(hier_cached_attention_fp8(q, c, odd), want)
        with pytest.raises(ValueError, match="mask list"):
            hier_cached_attention_fp8(q, c, dataclasses.replace(tiles, kv_mask=shifted(tiles.kv_mask)))


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("size,scale", [(1.0, 1e9), (1.0, 1e20), (1.0, 1e30), (1e30, 0.125), (1e30, 1e6)])
@pytest.mark.parametrize("case", [CASES[0], CASES[1], CASES[2]], ids=lambda c: c[0])
def test_scores_of_any_magnitude(case, size, scale, splits, monkeypatch):
    """Scores far from 0 on either side, also below any start that a running max
    could have: the largest takes all the weight, equal ones share it.  One channel
    of a query is not 0 and k is positive there, so that a score is one product
    (12 bits, exact) and unequal ones differ by 2^-4 of them or more: the weights
    are those of the formula, whatever the arithmetic.  lse: the scale times
    log2 e and its way back, the product and the sum round by 2^-24 of it each."""
    need_gpu()
    monkeypatch.setattr(kernels, "_fp8_splits", lambda workgroups, max_tiles: splits)

    def positive(c, f, k, v):
        k[:, :, 0] = k[:, :, 0].abs() + 0.25

    c, q, tiles = _rollout(case, seed=6, hide=positive)
    sign = torch.where(torch.arange(q.shape[0], device="cuda") % 3 == 0, -1.0, 1.0)
    q[:, :, 1:] = 0
    q[:, :, 0] = ((q[:, :, 0].float().abs() + 0.25).double() * size * sign[:, None]).to(torch.bfloat16)
    say("fp8 scores", case[0], size, scale, splits)
    lse = torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")
    out = hier_cached_attention_fp8(q, c, tiles, lse=lse, scale=scale)
    torch.cuda.synchronize()
    ref, bound, rlse = _reference(q, c, tiles, scale)
    assert bool(((out.double() - ref).abs() <= bound).all())
    some = ~torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse), ~some)
    assert bool(((lse.double() - rlse).abs() <= STEP + 2.0 ** -21 * rlse.abs())[some].all())


def test_the_normaliser_of_rows_that_are_not_numbers():
    """lse is NaN where the output is (-inf is a row that sees no key)."""
    need_gpu()
    for case in (CASES[0], CASES[2], CASES[4]):
        c, q, tiles = _rollout(case)
        q[1, q.shape[1] - 1, 3] = float("nan")
        lse = torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")
        for splits in (1, 2):
            with pytest.MonkeyPatch.context() as m:
                m.setattr(kernels, "_fp8_splits", lambda workgroups, max_tiles: splits)
                out = hier_cached_attention_fp8(q, c, tiles, lse=lse)
            assert bool(torch.isnan(out[1, -1]).all())
            assert torch.equal(torch.isnan(lse), torch.isnan(out).all(-1).t()), case[0]


@pytest.mark.parametrize("dtype", [FP8, torch.bfloat16])
def test_a_cache_keeps_the_device_that_its_pools_are_on(dtype):
    """Made on "cuda", without an index: row tables of later appends go to the
    pools' device, not to the one that is current then."""
    need_gpu()
    c = _cache(dtype=dtype)
    assert c.device == c.k.device and c.device.index is not None
    blk = torch.zeros(_rows(c, 2), 3, 64, dtype=torch.bfloat16, device="cuda")
    c.append(blk, blk, 0, 2, [[True, True]] * 2)
    assert all(t.device == c.k.device for t in c._dst_cache.values())
