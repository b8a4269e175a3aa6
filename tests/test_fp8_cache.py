"""CPU checks of the 8-bit paged cache: its pages and block tables, the values
it stands for, and what it refuses."""

import numpy as np
import pytest
import torch

from multics_amd import metadata as M
from multics_amd.kernels import (hier_attention_forward, hier_cached_attention_fp8,
                                 qk_head_prologue)
from multics_amd.module import SelfAttention
from multics_amd.paged_cache import HierPagedKVCache

FP8 = torch.float8_e4m3fn


def _cache(dtype=FP8, L=37, KL=3, KG=18, no_local=False, **kw):
    return HierPagedKVCache(**{**dict(
        num_players=3, num_groups=0 if no_local else 2, num_patches=L,
        num_local_hub_tokens=0 if no_local else KL, num_global_hub_tokens=KG, num_heads=2,
        head_dim=64, local_attn_size=4, num_frame_per_block=2, device="cpu", dtype=dtype,
        hier_no_local_hub=no_local), **kw})


@pytest.mark.parametrize("no_local", [False, True])
@pytest.mark.parametrize("L,KL,KG", [(37, 3, 18), (16, 16, 1), (1, 1, 1), (33, 5, 6)])
def test_blocks_cover_the_tokens_and_stay_in_their_pages(L, KL, KG, no_local):
    c = _cache(L=L, KL=KL, KG=KG, no_local=no_local)
    assert all(p % 16 == 0 for p in c.pages) and c.k.shape[0] % 16 == 0
    assert c.k_scale.shape == (c.k.shape[0] // 16, 2)
    pages = {}
    for f in range(c.R):
        rows, table = c.block_rows(f, 1), c.block_table(f, 1)
        assert table[:, 2].min() >= 1 and table[:, 2].max() <= 16
        assert (table[:, 1] % 16 == 0).all()
        src = np.concatenate([s + np.arange(n) for s, _, n in table])
        dst = np.concatenate([d + np.arange(n) for _, d, n in table])
        assert np.array_equal(src, np.arange(len(rows))) and np.array_equal(dst, rows)
        for d in table[:, 1]:                    # a block of 16 belongs to one frame only
            assert pages.setdefault(int(d), f) == f
    assert sorted(pages) == list(range(0, c.k.shape[0], 16))
    wrap = c.block_table(c.R - 1, 2)             # a block over the ring's end
    assert np.array_equal(np.concatenate([d + np.arange(n) for _, d, n in wrap]),
                          c.block_rows(c.R - 1, 2))


def test_the_bf16_cache_keeps_its_pages():
    c = _cache(torch.bfloat16)
    assert c.pages == (37, 3, 18) and c.k_scale is None and not c.fp8
    assert c.dequantised()[0] is c.k


def test_values_are_codes_times_scales():
    c = _cache()
    assert torch.count_nonzero(c.dequantised()[0]) == 0
    c.k[5, 1] = torch.tensor(1.75).to(FP8)
    c.k_scale[0, 1] = torch.tensor(2.0 ** -100).to(torch.float8_e8m0fnu)
    c.v[17, 0] = torch.tensor(-448.0).to(FP8)
    c.v_scale[1, 0] = torch.tensor(2.0 ** 119).to(torch.float8_e8m0fnu)
    k, v = c.dequantised()
    assert k.dtype == torch.bfloat16 and float(k[5, 1, 3].double()) == 1.75 * 2.0 ** -100
    assert float(v[17, 0, 9].double()) == -448 * 2.0 ** 119


def test_window_lists_of_the_two_caches_are_kept_apart(monkeypatch):
    """Equal windows of a bf16 and an 8-bit cache lie at different rows."""
    from types import SimpleNamespace
    built = []
    monkeypatch.setattr(M, "build", lambda topo, device: SimpleNamespace(
        tiles=built.append(topo) or SimpleNamespace()))
    monkeypatch.setattr(M, "_META_CACHE", type(M._META_CACHE)())
    lists = []
    for c in (_cache(torch.bfloat16), _cache()):
        for f in range(4):
            c.slot_frame[f] = f
            c.local_active[:, f] = True
        kw = dict(device="cpu", n_frames=2, n_block=2, local_attn=4,
                  labels=np.zeros((2, 3), np.int64), q_active=np.ones((2, 2), bool),
                  direct_player=True)
        lists.append(M.cached_window_tiles(c, 3, **kw))
        assert M.cached_window_tiles(c, 3, **kw) is lists[-1]
    assert lists[0] is not lists[1] and len(built) == 2
    assert built[0].tile_agent_base != built[1].tile_agent_base


def test_refusals():
    with pytest.raises(NotImplementedError, match="head_dim"):
        _cache(head_dim=32)
    with pytest.raises(NotImplementedError, match="float8_e4m3fn"):
        _cache(torch.float8_e5m2)
    c = _cache(local_attn_size=-1, max_frames=4)
    S = 3 * 2 * 37 + 2 * (2 * 3 + 18)
    blk = torch.zeros(S, 2, 64, dtype=torch.bfloat16)
    act = np.ones((2, 2), bool)
    with pytest.raises(ValueError, match="bf16"):
        c.append(blk.float(), blk.float(), 0, 2, act)
    with pytest.raises(ValueError, match="must be"):
        c.append(blk[:-1], blk[:-1], 0, 2, act)
    with pytest.raises(ValueError, match="max_frames"):
        c.append(blk, blk, 3, 2, act)
    with pytest.raises(ValueError, match="GPU"):
        c.append(blk, blk, 0, 2, act)            # no kernel takes host memory
    assert (c.slot_frame == -1).all()
    q = torch.zeros(S, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="inference-only"):
        hier_cached_attention_fp8(q.clone().requires_grad_(), c, None)
    with pytest.raises(ValueError, match="not held in 8 bits"):
        hier_cached_attention_fp8(q, _cache(torch.bfloat16), None)
    with pytest.raises(NotImplementedError, match="GPU"):
        hier_cached_attention_fp8(q, c, None)
    with pytest.raises(NotImplementedError, match="bf16"):
        hier_cached_attention_fp8(q.float(), c, None)
    with pytest.raises(NotImplementedError):
        hier_attention_forward(q, c.k, c.v, None, q)
    with pytest.raises(ValueError, match="qk_norm"):
        SelfAttention(128, 2, qk_norm="heads")
    with pytest.raises(NotImplementedError, match="GPU"):
        qk_head_prologue(q.view(S, 128), q.view(S, 128), norm_q_w=torch.ones(64),
                         norm_k_w=torch.ones(64), rope_cos=torch.ones(S, 32),
                         rope_sin=torch.zeros(S, 32), num_heads=2, eps=1e-6)


def test_per_head_norm_on_the_host():
    """The torch tail (any device) norms each head by itself."""
    torch.manual_seed(1)
    m = SelfAttention(256, 4, qk_norm="head")
    torch.nn.init.normal_(m.norm_q.weight)
    x = torch.randn(1, 6, 256)
    q, _, _ = m._project_self_attn_qkv(x, torch.ones(6, 1, 32, dtype=torch.complex128))
    h = m.q(x).double().view(6, 4, 64)
    ref = h / torch.sqrt(h.square().mean(-1, keepdim=True) + m.eps) * m.norm_q.weight.double()
    assert torch.allclose(q.double().view(6, 4, 64), ref, rtol=1e-5, atol=1e-6)
    assert SelfAttention(256, 4).norm_q.weight.shape == (256,)


def test_struct_layouts_match_c(tmp_path, monkeypatch):
    from multics_amd import _capi
    from tests import test_capi
    monkeypatch.setattr(test_capi, "STRUCTS", {
        n: getattr(_capi, n) for n in ("HierHeadNormArgs", "HierHeadNormBwdArgs", "HierPageFp8Args",
                                       "HierFwdFp8Args")})
    test_capi.test_ctypes_struct_layout_matches_c(tmp_path)


def test_c_entries_refuse_before_a_launch():
    """Bad sizes, pointers and strides of the C calls: an error each, and no
    launch (made-up addresses, never read)."""
    from multics_amd import _capi
    lib, at = _capi.lib(), 0x7f0000000000
    EINVAL, EUNSUP = _capi.HIER_EINVAL, _capi.HIER_EUNSUPPORTED
    import ctypes as C

    def fill(cls, **kw):
        a = cls()
        for i, (name, t) in enumerate(cls._fields_):
            setattr(a, name, at + 4096 * i if t is _capi.vp else 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    good = {
        "hier_head_prologue": (_capi.HierHeadNormArgs, dict(S=4, Hq=2, Hk=1, D=64, eps=1e-6)),
        "hier_head_prologue_bwd": (_capi.HierHeadNormBwdArgs,
                                   dict(S=4, Hq=2, Hk=1, D=64, eps=1e-6, partial_rows=2)),
        "hier_kv_append_fp8": (_capi.HierPageFp8Args, dict(H=2, D=64, n_blocks=1, n_rows=4,
                                                           pool_rows=64)),
        "hier_attn_fwd_fp8": (_capi.HierFwdFp8Args, dict(H=4, Hk=2, D=128, n_items=3, scale=1.0,
                                                         splits=2, kv_rows=64, q_rows=8)),
    }
    bad = {
        "hier_head_prologue": [(dict(D=96), EUNSUP), (dict(Hq=0), EINVAL), (dict(S=-1), EINVAL),
                               (dict(qx=0), EINVAL), (dict(kx=at + 8), EINVAL),
                               (dict(qx_ss=7), EINVAL), (dict(S=1 << 33), EUNSUP)],
        "hier_head_prologue_bwd": [(dict(D=32), EUNSUP), (dict(S=0), EINVAL), (dict(dq=0), EINVAL),
                                   (dict(dk_sh=4), EINVAL), (dict(partial_rows=1), EINVAL),
                                   (dict(S=100), EINVAL)],
        "hier_kv_append_fp8": [(dict(D=80), EUNSUP), (dict(pool_rows=40), EINVAL),
                               (dict(blocks=0), EINVAL), (dict(k_pool=at + 1), EINVAL),
                               (dict(v_src_ss=3), EINVAL), (dict(pool_ss=8), EINVAL),
                               (dict(n_blocks=1 << 30), EUNSUP)],
        "hier_attn_fwd_fp8": [(dict(D=256), EUNSUP), (dict(H=3), EINVAL), (dict(splits=0), EINVAL),
                              (dict(splits=33), EINVAL), (dict(part_o=0), EINVAL),
                              (dict(scale=0.0), EINVAL), (dict(v_scale=0), EINVAL),
                              (dict(kv_ss=8), EINVAL), (dict(kv_rows=1 << 25), EUNSUP),
                              (dict(kv_rows=1 << 24, kv_ss=1024), EUNSUP),
                              (dict(kv_rows=1 << 24, scale_ss=8192), EUNSUP),
                              (dict(n_items=1 << 24), EUNSUP)],
    }
    for name, cases in bad.items():
        cls, base = good[name]
        assert getattr(lib, name)(None, None) == EINVAL
        for change, want in cases:
            assert getattr(lib, name)(C.byref(fill(cls, **{**base, **change})), None) == want, \
                (name, change, lib.hier_last_error())
            assert lib.hier_last_error()
    # nothing to do is no error, whatever the rest holds
    assert lib.hier_head_prologue(C.byref(fill(_capi.HierHeadNormArgs, S=0, Hq=1, Hk=1, D=64)), None) == 0
    assert lib.hier_kv_append_fp8(C.byref(fill(_capi.HierPageFp8Args, H=1, D=64)), None) == 0
    assert lib.hier_attn_fwd_fp8(C.byref(fill(_capi.HierFwdFp8Args, H=1, Hk=1, D=64, splits=1)), None) == 0


def test_packed_arguments_are_the_structures():
    from multics_amd import _capi
    import ctypes as C
    for cls in (_capi.HierHeadNormArgs, _capi.HierHeadNormBwdArgs, _capi.HierPageFp8Args,
                _capi.HierFwdFp8Args):
        vals = [0.5 if t is _capi.f32 else 3 + 7 * i for i, (_, t) in enumerate(cls._fields_)]
        a = cls.from_buffer_copy(_capi.packer(cls)(*vals))
        assert [getattr(a, n) for n, _ in cls._fields_] == vals


def _refused(name, cls, base, bad):
    """Every change of ``base`` (sizes; made-up addresses, never read) is refused."""
    import ctypes as C
    from multics_amd import _capi
    for change in bad:
        a = cls()
        for i, (field, t) in enumerate(cls._fields_):
            setattr(a, field, 0x7f0000000000 + 4096 * i if t is _capi.vp else 0)
        for field, value in {**base, **change}.items():
            setattr(a, field, value)
        assert getattr(_capi.lib(), name)(C.byref(a), None) in (
            _capi.HIER_EINVAL, _capi.HIER_EUNSUPPORTED), (name, change)
    # (an empty call clears the message)
    assert _capi.lib().hier_kv_append_fp8(C.byref(_capi.HierPageFp8Args(H=1, D=64)), None) == 0


def test_c_norms_refuse_an_eps_below_0():
    from multics_amd import _capi
    bad = [dict(eps=x) for x in (-1e-6, -1.0, float("nan"), float("inf"), float("-inf"))]
    size = dict(S=4, Hq=2, Hk=1, D=64, partial_rows=2)
    _refused("hier_head_prologue_bwd", _capi.HierHeadNormBwdArgs, size, bad)
    size.pop("partial_rows")
    _refused("hier_head_prologue", _capi.HierHeadNormArgs, size, bad)


def test_c_attention_refuses_lists_that_it_cannot_read_whole():
    """Masks are read 16 bytes at a time, row-table entries 8."""
    from multics_amd import _capi
    at = 0x7f0000000000
    size = dict(H=4, Hk=2, D=128, n_items=3, scale=1.0, splits=2, kv_rows=64, q_rows=8)
    _refused("hier_attn_fwd_fp8", _capi.HierFwdFp8Args, size,
             [dict(tile_kv_mask=at + 4), dict(tile_kv_mask=at + 8), dict(row_table=at + 4)])


def test_c_attention_refuses_a_scale_that_is_not_a_number():
    from multics_amd import _capi
    size = dict(H=4, Hk=2, D=128, n_items=3, splits=2, kv_rows=64, q_rows=8)
    _refused("hier_attn_fwd_fp8", _capi.HierFwdFp8Args, size,
             [dict(scale=x) for x in (float("nan"), float("inf"), 2e30, -1.0, 0.0)])


def test_c_attention_refuses_a_grid_of_2_32_threads():
    """2^24 workgroups of 256, reached by rounding up to the number of XCDs too."""
    from multics_amd import _capi
    size = dict(H=1, Hk=1, D=64, scale=1.0, splits=1, kv_rows=64, q_rows=8)
    _refused("hier_attn_fwd_fp8", _capi.HierFwdFp8Args, size,
             [dict(n_items=(1 << 24) - i) for i in (0, 1, 7)] + [dict(n_items=(1 << 23) - 1, splits=2)])


def test_list_offsets_are_refused_past_31_bits():
    assert M._list_offsets([64, 0, 128]).tolist() == [0, 64, 64, 192]
    most = (1 << 31) - 64
    assert int(M._list_offsets([most - 64, 64])[-1]) == most
    for lengths in ([most, 64], np.full(5, 1 << 30, np.int32), [1 << 31]):
        with pytest.raises(NotImplementedError, match="entries"):
            M._list_offsets(lengths)
