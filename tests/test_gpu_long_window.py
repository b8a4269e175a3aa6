"""Tile lists of cached windows of more frames, or more tokens, than the
builder's arrays in LDS hold (1,024 runs of frames, 262,144 slots a stream)."""

import numpy as np
import pytest

from multics_amd import metadata as M
from tests.gpu_util import expand_tiles, need_gpu, say

pytestmark = pytest.mark.gpu


def _window(P, N, L, KL, KG, n, W, frames, labels):
    """List of the block that ends a window of ``frames``; frame f's rows of a
    stream lie at its base + 32 f (pages with a gap)."""
    pitch = -(-max(L, KL, KG) // 16) * 16 + 16
    base = lambda s: [(s * frames + f) * pitch for f in range(frames)]  # noqa: E731
    bases = ([base(p) for p in range(P)], [base(P + g) for g in range(N)], base(P + N))
    act = [[g in labels for g in range(N)]] * n
    topo = M.cached_topology(
        P=P, N=N, L=L, KL=KL, KG=KG, n_frames=n, n_block=n, local_attn=W,
        agent_frame_lists=[list(range(frames))] * P, local_frame_lists=[list(range(frames))] * N,
        global_frame_list=list(range(frames)),
        local_active_frames=[[act[0][g]] * frames for g in range(N)], labels=[labels] * n,
        q_active=act, direct_player=True, tile_bases=bases)
    return topo, bases


def _expected(P, N, L, KL, KG, n, W, frames, labels, bases):
    """{row: keys} from the rules of a window, frame by frame."""
    rows, width = {}, (L, KL, KG)
    keys = lambda kind, s, f: range((bases[kind][s] if kind < 2 else bases[2])[f],  # noqa: E731
                                    (bases[kind][s] if kind < 2 else bases[2])[f] + width[kind])
    span = lambda kind, s, fs: [k for f in fs for k in keys(kind, s, f)]  # noqa: E731
    for j in range(n):
        f = frames - n + j
        near = [x for x in range(frames) if f - x < W]
        now = range(frames - n, frames)
        for p in range(P):
            seen = set(span(0, p, near) + span(1, labels[p], near))
            for o in range(P):
                if o != p and labels[o] == labels[p]:
                    seen |= set(span(0, o, now))
            for i in range(L):
                rows[(p * n + j) * L + i] = seen
        for g in range(N):
            if g in labels:
                seen = set(span(1, g, near) + span(2, 0, near))
                for p in range(P):
                    if labels[p] == g:
                        seen |= set(span(0, p, near))
                for i in range(KL):
                    rows[P * n * L + (j * N + g) * KL + i] = seen
            else:
                for i in range(KL):
                    rows[P * n * L + (j * N + g) * KL + i] = set()
        seen = set(span(2, 0, near))
        for g in set(labels):
            seen |= set(span(1, g, near))
        for i in range(KG):
            rows[P * n * L + n * N * KL + j * KG + i] = seen
    return rows


@pytest.mark.parametrize("shape", [
    (1, 1, 2, 1, 1, 1, 699, 700, [0]),            # 2,100 runs
    (2, 2, 3, 2, 1, 2, 500, 1100, [0, 0]),        # a window inside, a group without members
    (3, 1, 1, 1, 2, 3, 340, 342, [0, 0, 0]),      # 1,374 runs: two chunks
    (1, 1, 941, 1, 1, 1, 299, 300, [0]),          # few runs, 282,000 slots
    (1, 1, 1, 1, 1, 1, 400, 341, [0]),            # 1,023 runs: the arrays hold them
])
def test_long_windows_list_the_rule(shape):
    need_gpu()
    say("long window", shape)
    topo, bases = _window(*shape)
    tiles = M.build(topo, "cuda").tiles
    want = _expected(*shape, bases)
    assert expand_tiles(tiles) == want
    assert tiles.logical_pairs == sum(len(v) for v in want.values())
    items = tiles.items.cpu().numpy()
    idx, mask = tiles.kv_idx.cpu().numpy(), tiles.kv_mask.cpu().numpy().view(np.uint32)
    both = tiles.blk_and.cpu().numpy().view(np.uint32)
    for it in items:
        off, cnt = it[5], it[6]
        assert cnt % 64 == 0 and tiles.max_keys >= cnt
        real = idx[off:off + cnt][mask[off:off + cnt] != 0]
        assert set(idx[off:off + cnt]) <= set(real) or len(real) == 0
        for k in range(cnt // 64):
            at = off + 64 * k
            assert both[at // 64] == np.bitwise_and.reduce(mask[at:at + 64])


def test_reference_formats_are_refused():
    need_gpu()
    topo, _ = _window(1, 1, 2, 1, 1, 1, 699, 700, [0])
    with pytest.raises(NotImplementedError, match="tile list only"):
        M.build(topo, "cuda", segmented_block_m=16)


def test_lists_past_31_bits_are_refused():
    """Four players' windows of 1.2e9 tokens: each stream's list fits, all of them
    together do not fit an item's offset.  Refused from the counts, before any list
    is made."""
    need_gpu()
    topo, _ = _window(4, 1, 1 << 18, 1, 1, 1, 1200, 1144, [0, 0, 0, 0])
    say("lists past 31 bits")
    with pytest.raises(NotImplementedError, match="2\\^31"):
        M.build(topo, "cuda")
