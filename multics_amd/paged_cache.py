"""Paged KV cache for the cached (chunked causal rollout) hierarchical attention.

The reference keeps one rolling buffer per stream -- P agent caches, N local
hub caches (+ per-token active flags), one global cache -- appends a block's
K/V, shifts the buffer when it overflows and concatenates every buffer into one
pool on each attention call (attention.py:90-228, 605-796;
wan_video_Nplayers.py:888-1058; hier_segmented_attention.py:458-469).

Here one layer owns a single K pool and a single V pool ``[rows, H, D]``.  Every
(stream, frame) has a fixed page of rows -- L rows for an agent frame, KL for a
local-hub frame, KG for a global frame -- in a ring of R = W + n frame slots
(W = local_attn_size, n = frames per block; R = max_frames when W = -1):

    rows [ agents p-major: P x R x L | locals g-major: N x R x KL | global: R x KG ]

Appending frame f writes slot f mod R of every stream with one HIP scatter
(``hier_kv_append``).  A re-run of the same block (a denoising step)
overwrites the same pages, which is the reference's refresh-in-place; a new
frame overwrites the page of frame f - R, which is the reference's eviction.
No row ever moves and nothing is concatenated: the attention tile list
addresses the pool rows directly.

With ``dtype=torch.float8_e4m3fn`` the pools hold 8-bit codes and, for every 16
rows and head, a power-of-two scale (``k_scale`` / ``v_scale``, e8m0
``[rows / 16, batch * H]``); a value is its code times its scale.  Pages are
padded to whole blocks of 16 rows, so that a block belongs to one page and is
always written as a whole (220 tokens: 224 rows; one token: 16, eight times
its bytes in bf16).  ``append`` quantises
(``hier_kv_append_fp8``), ``kernels.hier_cached_attention_fp8`` reads the codes.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np
import torch

from . import _capi


_stream = _capi.stream_of

FP8_BLOCK = 16      # rows that share a scale (HIER_FP8_BLOCK)
_pack_page = _capi.packer(_capi.HierPageFp8Args)


class HierPagedKVCache:
    """One layer's hierarchical KV cache (pools + ring bookkeeping).

    Reads like the reference's cache dict for the keys the attention module
    inspects (``hier_hub``, ``num_players``, ``num_groups``,
    ``num_local_hub_tokens``, ``num_global_hub_tokens``, ``hier_no_local_hub``).

    ``batch`` > 1 holds that many caches of the same topology in one pool,
    interleaved per row: ``k`` / ``v`` are ``[rows, batch * H, D]``, so batch
    member b's head h is head ``b * H + h``.  The classifier-free-guidance
    pair of caches (wan_video_Nplayers.py:645-648, one model call per prompt
    at :739-776) then shares the ring bookkeeping, the tile list and one
    kernel launch per block, which sees ``batch * H`` heads.

    ``dtype`` is bf16, or ``torch.float8_e4m3fn`` for a cache held in 8 bits
    (head dim 64 or 128).  Its pages are whole blocks of 16 rows of a byte a
    channel and the scales: half of bf16's memory for frames of many tokens
    (220: 0.51), as much for pages of eight, more for smaller ones (six tokens:
    1.3 times, five: 1.6, one: 8).
    """

    def __init__(self, *, num_players: int, num_groups: int, num_patches: int,
                 num_local_hub_tokens: int, num_global_hub_tokens: int, num_heads: int,
                 head_dim: int, local_attn_size: int, num_frame_per_block: int, device,
                 dtype=torch.bfloat16, max_frames: Optional[int] = None,
                 hier_no_local_hub: bool = False, batch: int = 1):
        self.P, self.N, self.L = int(num_players), int(num_groups), int(num_patches)
        self.KL, self.KG = int(num_local_hub_tokens), int(num_global_hub_tokens)
        self.H, self.D = int(num_heads), int(head_dim)
        self.B = int(batch)
        if self.B < 1:
            raise ValueError(f"batch must be >= 1, got {batch}")
        self.W, self.n = int(local_attn_size), int(num_frame_per_block)
        self.no_local = bool(hier_no_local_hub)
        if self.no_local and (self.KL != 0 or self.KG <= 0):
            raise ValueError("hier_no_local_hub requires K_L=0 and K_G>0")
        if self.W == -1:
            if max_frames is None:
                raise ValueError("an unbounded window (local_attn_size=-1) needs max_frames")
            self.R = int(max_frames)
        else:
            if self.W < self.n:
                raise ValueError("hier_hub requires local_attn_size=-1 or >= num_frame_per_block")
            self.R = self.W + self.n
        self.fp8 = dtype == torch.float8_e4m3fn
        if dtype.itemsize == 1 and not self.fp8:
            raise NotImplementedError(f"an 8-bit cache holds float8_e4m3fn, got {dtype}")
        if self.fp8 and self.D not in (64, 128):
            raise NotImplementedError(f"an 8-bit cache supports head_dim 64/128, got {self.D}")
        # rows of a page: the frame's tokens, in whole blocks when they share scales
        page = (lambda w: -(-w // FP8_BLOCK) * FP8_BLOCK) if self.fp8 else (lambda w: w)
        self.pages = (page(self.L), page(self.KL), page(self.KG))
        self.a_rows = self.P * self.R * self.pages[0]
        self.l_rows = 0 if self.no_local else self.N * self.R * self.pages[1]
        self.g_rows = self.R * self.pages[2]
        rows = self.a_rows + self.l_rows + self.g_rows
        self.device = torch.device(device)
        heads = self.B * self.H
        if self.fp8:
            # head-major storage: a head's codes of a page lie in one piece
            code = lambda: torch.zeros((heads, rows, self.D), dtype=torch.uint8,  # noqa: E731
                                       device=self.device).view(dtype).transpose(0, 1)
            one = lambda: torch.full((heads, rows // FP8_BLOCK), 127, dtype=torch.uint8,  # noqa: E731
                                     device=self.device).view(torch.float8_e8m0fnu).t()
            self.k, self.v, self.k_scale, self.v_scale = code(), code(), one(), one()
        else:
            self.k = torch.zeros((rows, heads, self.D), dtype=dtype, device=self.device)
            self.v = torch.zeros_like(self.k)
            self.k_scale = self.v_scale = None
        # the pools' own device, whichever is current at an append ("cuda" alone
        # would send the row tables to the device that is current then)
        self.device = self.k.device
        self.slot_frame = np.full(self.R, -1, dtype=np.int64)
        self.local_active = np.zeros((max(self.N, 1), self.R), dtype=bool)
        self._dst_cache = {}

    # ---- the reference dict contract (read-only) -------------------------------

    def _meta(self):
        return {"hier_hub": True, "num_players": self.P, "num_groups": self.N,
                "num_local_hub_tokens": self.KL, "num_global_hub_tokens": self.KG,
                "hier_no_local_hub": self.no_local}

    def __getitem__(self, key):
        return self._meta()[key]

    def get(self, key, default=None):
        return self._meta().get(key, default)

    def reset(self):
        """Forget every cached frame (wan_video_Nplayers.py:1024-1058)."""
        self.slot_frame.fill(-1)
        self.local_active.fill(False)

    # ---- addressing ----------------------------------------------------------------

    def agent_row(self, p: int, frame):
        """First pool row of a frame's page (or of each of an array of frames)."""
        return (p * self.R + frame % self.R) * self.pages[0]

    def local_row(self, g: int, frame):
        return self.a_rows + (g * self.R + frame % self.R) * self.pages[1]

    def global_row(self, frame):
        return self.a_rows + self.l_rows + (frame % self.R) * self.pages[2]

    def block_rows(self, start_frame: int, n: int) -> np.ndarray:
        """Pool row of every token of a block in the cached query order
        [P*n*L agents | n*N*KL locals | n*KG global]."""
        P, N, L, KL, KG = self.P, self.N, self.L, self.KL, self.KG
        pa, pl, pg = self.pages
        fr = start_frame + np.arange(n)
        slot = fr % self.R
        agent = ((np.arange(P)[:, None, None] * self.R + slot[None, :, None]) * pa +
                 np.arange(L)[None, None, :]).reshape(-1)
        local = (self.a_rows + (np.arange(N)[None, :, None] * self.R + slot[:, None, None]) * pl +
                 np.arange(KL)[None, None, :]).reshape(-1) if not self.no_local else \
            np.zeros(0, np.int64)
        glob = (self.a_rows + self.l_rows + slot[:, None] * pg + np.arange(KG)[None, :]).reshape(-1)
        return np.concatenate([agent, local, glob]).astype(np.int32)

    def block_table(self, start_frame: int, n: int) -> np.ndarray:
        """``[n_blocks, 3]`` int32 (source row, pool row, rows) of the blocks of
        16 pool rows that a block's tokens fill: every page's tokens in runs
        of 16, the last shorter."""
        rows = self.block_rows(start_frame, n)
        src, count, at = [], [], 0
        for pages, width in ((self.P * n, self.L), (0 if self.no_local else n * self.N, self.KL),
                             (n, self.KG)):
            first = np.arange(0, width, FP8_BLOCK)
            src.append((at + np.arange(pages)[:, None] * width + first).reshape(-1))
            count.append(np.tile(np.minimum(FP8_BLOCK, width - first), pages))
            at += pages * width
        src = np.concatenate(src)
        return np.stack([src, rows[src], np.concatenate(count)], axis=1).astype(np.int32)

    # ---- append ----------------------------------------------------------------------

    def append(self, k_blk: torch.Tensor, v_blk: torch.Tensor, start_frame: int, n: int,
               active_block) -> None:
        """Write a block's roped K and V ``[S_blk, batch * H, D]`` (cached
        order; batch-major heads) into the pages of frames [start_frame,
        start_frame + n); ``active_block`` [n, N] are the local-hub slot flags
        of those frames."""
        S = self.P * n * self.L + n * ((0 if self.no_local else self.N * self.KL) + self.KG)
        HB = self.B * self.H
        if k_blk.shape != (S, HB, self.D) or v_blk.shape != (S, HB, self.D):
            raise ValueError(f"block K/V must be [{S}, {HB}, {self.D}], "
                             f"got {tuple(k_blk.shape)}, {tuple(v_blk.shape)}")
        want = torch.bfloat16 if self.fp8 else self.k.dtype
        if k_blk.dtype != want or v_blk.dtype != want:
            raise ValueError("block K/V dtype must match the cache" if not self.fp8 else
                             "an 8-bit cache takes bf16 K/V")
        if self.fp8 and (k_blk.device != self.k.device or v_blk.device != self.k.device):
            raise ValueError(f"block K/V must be on the cache's device {self.k.device}")
        if n > self.R:
            raise ValueError(f"a block of {n} frames does not fit a window of {self.R} frames")
        if self.W == -1 and (start_frame < 0 or start_frame + n > self.R):
            # an unbounded window keeps every frame: a ring slot may never be
            # reused, or the window would silently lose its oldest frames
            raise ValueError(f"frames [{start_frame}, {start_frame + n}) exceed the cache's "
                             f"max_frames={self.R} (local_attn_size=-1 keeps every frame)")
        key = (start_frame % self.R, n)
        dst = self._dst_cache.get(key)
        if dst is None:
            dst = torch.from_numpy(self.block_table(start_frame, n) if self.fp8 else
                                   self.block_rows(start_frame, n)).to(self.device)
            self._dst_cache[key] = dst
        if self.fp8:
            self._append_fp8(k_blk, v_blk, dst)
        else:
            self._append_rows(k_blk, v_blk, dst)
        act = np.asarray(active_block, dtype=bool).reshape(n, -1)
        for j in range(n):
            slot = (start_frame + j) % self.R
            self.slot_frame[slot] = start_frame + j
            if not self.no_local:
                self.local_active[:, slot] = act[j, :self.N]

    def _append_rows(self, k_blk, v_blk, dst) -> None:
        S, HB = k_blk.shape[:2]
        if k_blk.stride(2) != 1 or v_blk.stride(2) != 1:
            k_blk, v_blk = k_blk.contiguous(), v_blk.contiguous()
        args = _capi.HierPageArgs(
            H=HB, D=self.D, n_rows=S, pool_rows=self.k.shape[0], k_src=k_blk.data_ptr(),
            v_src=v_blk.data_ptr(), k_src_ss=k_blk.stride(0), k_src_sh=k_blk.stride(1),
            v_src_ss=v_blk.stride(0), v_src_sh=v_blk.stride(1), dst_rows=dst.data_ptr(),
            k_pool=self.k.data_ptr(), v_pool=self.v.data_ptr(), pool_ss=self.k.stride(0),
            pool_sh=self.k.stride(1))
        _capi.call("hier_kv_append", C.byref(args), _stream(self.device))

    def _append_fp8(self, k_blk, v_blk, blocks) -> None:
        k, k_ss, k_sh = _capi.head_strides(k_blk)
        v, v_ss, v_sh = _capi.head_strides(v_blk)
        k_pool, v_pool, k_scale, v_scale, pool_ss, pool_sh, scale_ss, scale_sh = self._pool
        _capi.call_on(self.k.device, "hier_kv_append_fp8", _pack_page(
            self.B * self.H, self.D, blocks.shape[0], k.shape[0], self.k.shape[0], k.data_ptr(),
            v.data_ptr(), k_ss, k_sh, v_ss, v_sh, blocks.data_ptr(), k_pool, v_pool, pool_ss, pool_sh,
            k_scale, v_scale, scale_ss, scale_sh))

    @property
    def _pool(self):
        """Addresses and strides of the 8-bit pools and their scales."""
        return (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                self.v_scale.data_ptr(), *self.k.stride()[:2], *self.k_scale.stride())

    def dequantised(self):
        """The ``(k, v)`` that an 8-bit cache stands for, bf16 ``[rows,
        batch * H, D]`` (exact: a code and a power of two fit a bf16)."""
        if not self.fp8:
            return self.k, self.v
        wide = lambda c, s: (c.float() * s.float().repeat_interleave(FP8_BLOCK, 0)[..., None]).to(  # noqa: E731
            torch.bfloat16)
        return wide(self.k, self.k_scale), wide(self.v, self.v_scale)

    # ---- window ----------------------------------------------------------------------

    def window(self, end_frame: int):
        """Frames held for a block ending at ``end_frame`` (the last R written
        frames up to it), their pool bases per stream and the local-hub active
        flag of each cached local frame."""
        f = self.slot_frame
        frames = np.sort(f[(f >= 0) & (f <= end_frame) & (f > end_frame - self.R)])
        groups = 0 if self.no_local else self.N
        agent = [self.agent_row(p, frames).tolist() for p in range(self.P)]
        local = [self.local_row(g, frames).tolist() for g in range(groups)]
        glob = self.global_row(frames).tolist() if self.KG > 0 else []
        lact = [self.local_active[g, frames % self.R].tolist() for g in range(groups)]
        return frames.tolist(), (agent, local, glob), lact


def init_hier_paged_kv_cache(*, num_layers: int, **kw):
    """One ``HierPagedKVCache`` per transformer layer (the reference allocates
    its per-layer stream dicts in wan_video_Nplayers.py:888-989)."""
    return [HierPagedKVCache(**kw) for _ in range(int(num_layers))]
