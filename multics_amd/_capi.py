"""ctypes binding of the C ABI in ``include/hierattn.h``.

The library is loaded from ``multics_amd/_lib/libhierattn.so`` (built in tree
by ``multics_amd.build``), or from the file named by ``HIERATTN_LIB``.  There is no fallback: when the library is missing
the import of a compute entry point raises.  Error codes map back to the
exception types the reference raises for the same conditions
(multics/models/kernels/hier_segmented_attention.py:425-431 NotImplementedError,
multics/models/attention.py:500-506 ValueError,
multics/models/kernels/hier_paged_attention.py:37-47 RuntimeError,
multics/models/kernels/hier_packed_attention.py:54-64 AssertionError).
"""

from __future__ import annotations

import ctypes as C
import os
import struct
import threading
from pathlib import Path

import torch

LIB_PATH = Path(os.environ.get("HIERATTN_LIB") or
                Path(__file__).resolve().parent / "_lib" / "libhierattn.so")

HIER_OK, HIER_EINVAL, HIER_EUNSUPPORTED, HIER_ELAUNCH, HIER_EINTERNAL = 0, -1, -2, -3, -4

i32, i64, f32, vp = C.c_int32, C.c_int64, C.c_float, C.c_void_p


class HierTopo(C.Structure):
    _fields_ = [(n, i32) for n in ("P", "N", "L", "KL", "KG", "n_frames", "n_block",
                                   "local_attn", "direct", "no_local", "use_membership", "B",
                                   "fa_max", "fl_max", "fg_max", "T_mem")] + \
               [(n, vp) for n in ("fa", "fl", "fg", "agent_frames", "local_frames",
                                  "global_frames", "local_active", "q_frames", "labels",
                                  "q_active", "membership", "global_only", "ref_agent_base",
                                  "ref_local_base", "ref_global_base", "tile_agent_base",
                                  "tile_local_base", "tile_global_base", "ref_qbase",
                                  "tile_qbase")] + \
               [("ref_qstride", i32 * 3), ("tile_qstride", i32 * 3)]


class HierMetaCounts(C.Structure):
    _fields_ = [(n, vp) for n in ("seg_count", "tiled_count", "dense_count", "logical_count",
                                  "tile_count")]


class HierMetaOut(C.Structure):
    _fields_ = [("block_m", i32)] + \
               [(n, vp) for n in ("seg_prog_off", "seg_kv_off", "seg_max_k", "seg_prog_qbase",
                                  "seg_prog_nq", "seg_prog_seg", "seg_kv_index", "seg_kv_count",
                                  "tiled_prog_off", "tiled_kv_off", "tiled_max_k",
                                  "tiled_prog_qbase", "tiled_prog_nq", "tiled_prog_seg",
                                  "tiled_kv_index", "tiled_kv_valid", "tiled_kv_count",
                                  "tile_kv_off", "tile_item_off")] + \
               [("rows_per_item", i32)] + \
               [(n, vp) for n in ("tile_kv_idx", "tile_kv_mask", "tile_blk_and", "tile_items")]


class HierPrologueArgs(C.Structure):
    _fields_ = [("S", i32), ("H", i32), ("D", i32), ("eps", f32)] + \
               [(n, vp) for n in ("qx", "kx", "vx", "cam", "w_cam_q", "w_cam_k")] + \
               [("C", i32)] + \
               [(n, vp) for n in ("norm_q_w", "norm_k_w", "rope_cos", "rope_sin", "q_out",
                                  "k_out", "v_out")] + \
               [("out_stride_s", i64), ("out_stride_h", i64)]


class HierFwdArgs(C.Structure):
    _fields_ = [("H", i32), ("D", i32), ("n_items", i32), ("scale", f32), ("kv_rows", i32),
                ("reserved", i32)] + \
               [(n, vp) for n in ("q", "k", "v", "o", "lse")] + \
               [(n, i64) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "v_ss", "v_sh", "o_ss", "o_sh",
                                   "lse_stride_h")] + \
               [(n, vp) for n in ("tile_items", "tile_kv_idx", "tile_kv_mask", "tile_blk_and",
                                  "row_table")]


class HierBwdArgs(C.Structure):
    _fields_ = [("H", i32), ("D", i32), ("n_items", i32), ("n_key_items", i32), ("scale", f32),
                ("kv_rows", i32), ("q_rows", i32), ("reserved", i32)] + \
               [(n, vp) for n in ("q", "k", "v", "o", "dout", "lse", "delta", "lse2", "dq", "dk",
                                  "dv")] + \
               [(n, i64) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "v_ss", "v_sh", "o_ss", "o_sh",
                                   "do_ss", "do_sh", "dq_ss", "dq_sh", "dk_ss", "dk_sh", "dv_ss",
                                   "dv_sh", "lse_stride_h")] + \
               [(n, vp) for n in ("tile_items", "tile_kv_idx", "tile_kv_mask", "tile_blk_and",
                                  "key_items", "key_q_idx", "key_q_mask", "key_blk_and")] + \
               [("n_ste_items", i32), ("ste_classes", i32)] + \
               [(n, vp) for n in ("ste_items", "ste_kv_idx", "ste_kv_mask", "ste_kv_class",
                                  "ste_partial")] + \
               [("ste_stride_h", i64), ("tile_kv_class", vp), ("tile_ste_first", vp),
                ("key_row_table", vp)]


class HierPageArgs(C.Structure):
    _fields_ = [("H", i32), ("D", i32), ("n_rows", i32), ("pool_rows", i32),
                ("k_src", vp), ("v_src", vp)] + \
               [(n, i64) for n in ("k_src_ss", "k_src_sh", "v_src_ss", "v_src_sh")] + \
               [("dst_rows", vp), ("k_pool", vp), ("v_pool", vp), ("pool_ss", i64),
                ("pool_sh", i64)]


class HierFrameAttnArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("B", "Lq", "Lk", "H", "D", "n_block", "local_attn")] + \
               [("scale", f32)] + [(n, vp) for n in ("q", "k", "v", "o")] + \
               [(n, i64) for n in ("q_sb", "q_ss", "q_sh", "k_sb", "k_ss", "k_sh", "v_sb", "v_ss",
                                   "v_sh", "o_sb", "o_ss", "o_sh")] + \
               [("q_frame", vp), ("k_frame", vp)]


class HierDeriveArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("n_items", "n_groups", "rows", "nq_max", "kv_len", "P", "T",
                                   "L", "N", "KL")] + \
               [(n, vp) for n in ("items", "kv_idx", "kv_mask", "ws")] + \
               [("ws_bytes", i64), ("totals", vp), ("key_entries", i64), ("ste_entries", i64)] + \
               [(n, vp) for n in ("key_items", "key_q_idx", "key_q_mask", "key_blk_and",
                                  "ste_items", "ste_kv_idx", "ste_kv_mask", "ste_blk_and",
                                  "ste_kv_class")]


class HierGateArgs(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("rows_per_gate", i32)] + \
               [(n, vp) for n in ("x", "y", "gate", "out")] + \
               [(n, i64) for n in ("x_ss", "y_ss", "gate_ss", "out_ss")]


class HierSteReduceArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("H", "P", "T", "L", "N", "KL", "classes")] + \
               [("partial", vp), ("stride_h", i64), ("out", vp)]


class HierMembershipArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("T", "N", "P", "B", "n", "fl_max")] + \
               [(n, vp) for n in ("logits", "la_frame", "membership", "global_only", "q_active",
                                  "local_active")]


class HierPrologueBwdArgs(C.Structure):
    _fields_ = [("S", i32), ("H", i32), ("D", i32), ("eps", f32), ("C", i32),
                ("tokens_per_wave", i32)] + \
               [(n, vp) for n in ("qx", "kx", "cam", "w_cam_q", "w_cam_k", "norm_q_w", "norm_k_w",
                                  "rope_cos", "rope_sin", "dq", "dk")] + \
               [(n, i64) for n in ("dq_ss", "dq_sh", "dk_ss", "dk_sh")] + \
               [(n, vp) for n in ("dqx", "dkx", "dw_q_partial", "dw_k_partial")]


class HierPrologueGradArgs(C.Structure):
    _fields_ = [(n, vp) for n in ("dnorm_q", "dnorm_k", "dw_cam_q", "dw_cam_k", "dwc_q_partial",
                                  "dwc_k_partial", "segments")]


class HierMergeArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("n_groups", "n_src", "rows", "rows_per_item")] + \
               [(n, vp) for n in ("items", "kv_idx", "kv_mask", "blk_and", "acc", "src_item",
                                  "src_group", "src_shift", "out_off", "out_cap", "group_desc",
                                  "group_item_off", "out_items", "src_from", "src_nbits")]


class HierTrimArgs(C.Structure):
    _fields_ = [("n_items", i32), ("reserved", i32)] + \
               [(n, vp) for n in ("items", "kv_mask", "row_table", "out_items")]


class HierHeadNormArgs(C.Structure):
    _fields_ = [("S", i64), ("Hq", i32), ("Hk", i32), ("D", i32), ("eps", f32),
                ("gain_bf16", i32), ("reserved", i32), ("qx", vp), ("kx", vp), ("qx_ss", i64), ("kx_ss", i64)] + \
               [(n, vp) for n in ("norm_q_w", "norm_k_w", "rope_cos", "rope_sin", "q_out",
                                  "k_out")] + \
               [(n, i64) for n in ("q_ss", "q_sh", "k_ss", "k_sh")]


class HierHeadNormBwdArgs(C.Structure):
    _fields_ = [("S", i64), ("Hq", i32), ("Hk", i32), ("D", i32), ("eps", f32),
                ("gain_bf16", i32), ("reserved", i32), ("qx", vp), ("kx", vp), ("qx_ss", i64), ("kx_ss", i64)] + \
               [(n, vp) for n in ("norm_q_w", "norm_k_w", "rope_cos", "rope_sin", "dq", "dk")] + \
               [(n, i64) for n in ("dq_ss", "dq_sh", "dk_ss", "dk_sh")] + \
               [(n, vp) for n in ("dqx", "dkx", "dnorm_q", "dnorm_k", "partial")] + \
               [("partial_rows", i64)]


class HierPageFp8Args(C.Structure):
    _fields_ = [("H", i32), ("D", i32), ("n_blocks", i32), ("n_rows", i32), ("pool_rows", i64),
                ("k_src", vp), ("v_src", vp)] + \
               [(n, i64) for n in ("k_src_ss", "k_src_sh", "v_src_ss", "v_src_sh")] + \
               [(n, vp) for n in ("blocks", "k_pool", "v_pool")] + \
               [("pool_ss", i64), ("pool_sh", i64), ("k_scale", vp), ("v_scale", vp),
                ("scale_ss", i64), ("scale_sh", i64)]


class HierFwdFp8Args(C.Structure):
    _fields_ = [(n, i32) for n in ("H", "Hk", "D", "n_items")] + \
               [("scale", f32), ("splits", i32), ("kv_rows", i64), ("q_rows", i64)] + \
               [(n, vp) for n in ("q", "k", "v", "k_scale", "v_scale", "o", "lse")] + \
               [(n, i64) for n in ("q_ss", "q_sh", "o_ss", "o_sh", "lse_stride_h", "kv_ss", "kv_sh",
                                   "scale_ss", "scale_sh")] + \
               [(n, vp) for n in ("tile_items", "tile_kv_idx", "tile_kv_mask", "tile_blk_and",
                                  "row_table", "part_o", "part_ml")]


class HierRmsNormArgs(C.Structure):
    _fields_ = [("M", i64), ("C", i32), ("eps", f32), ("type", i32), ("gain_type", i32)] + \
               [(n, vp) for n in ("x", "r", "w", "y", "h")] + \
               [(n, i64) for n in ("x_ss", "r_ss", "y_ss", "h_ss")]


class HierRmsNormBwdArgs(C.Structure):
    _fields_ = [("M", i64), ("C", i32), ("eps", f32), ("type", i32), ("gain_type", i32)] + \
               [(n, vp) for n in ("x", "r", "w", "dy", "dh", "dx", "dw", "partial")] + \
               [(n, i64) for n in ("x_ss", "r_ss", "dy_ss", "dh_ss", "dx_ss", "partial_rows")]


class HierLinearArgs(C.Structure):
    _fields_ = [("M", i64)] + [(n, i32) for n in ("N", "K", "type", "act")] + \
               [(n, vp) for n in ("x", "w", "bias", "residual", "gate", "out", "preact")] + \
               [(n, i64) for n in ("x_ss", "w_ss", "residual_ss", "gate_ss", "out_ss", "preact_ss",
                                   "rows_per_gate")] + \
               [("workspace", vp), ("workspace_bytes", i64)]


class HierPadRowsArgs(C.Structure):
    _fields_ = [(n, i64) for n in ("rows0", "rows1", "ss0", "ss1")] + \
               [(n, vp) for n in ("src0", "src1", "dst0", "dst1")] + [("C", i32), ("pad", i32)]   # the header's pairs


class HierLinearBwdArgs(C.Structure):
    _fields_ = [("M", i64)] + [(n, i32) for n in ("N", "K", "type", "act")] + \
               [(n, vp) for n in ("x", "w", "gate", "dy", "preact", "dx", "dw", "db", "dgate")] + \
               [(n, i64) for n in ("x_ss", "w_ss", "gate_ss", "dy_ss", "preact_ss", "dx_ss", "dw_ss",
                                   "rows_per_gate")] + \
               [("workspace", vp), ("workspace_bytes", i64)]


class HierCrossArgs(C.Structure):
    _fields_ = [(n, i32) for n in ("B", "Hq", "Hk", "D", "type")] + \
               [("scale", f32), ("Sq", i64), ("Sk", i64)] + \
               [(n, vp) for n in ("q", "k", "v", "o", "lse", "kv_lens", "key_mask")] + \
               [(n, i64) for n in ("q_sb", "q_ss", "q_sh", "k_sb", "k_ss", "k_sh", "v_sb", "v_ss", "v_sh",
                                   "o_sb", "o_ss", "o_sh", "mask_sb")] + \
               [("workspace", vp), ("workspace_bytes", i64)]


class HierCrossBwdArgs(C.Structure):
    _fields_ = [("f", HierCrossArgs)] + [(n, vp) for n in ("dout", "dq", "dk", "dv")] + \
               [(n, i64) for n in ("do_sb", "do_ss", "do_sh", "dq_sb", "dq_ss", "dq_sh", "dk_sb", "dk_ss",
                                   "dk_sh", "dv_sb", "dv_ss", "dv_sh")]


def _formats(cls) -> str:
    codes = {i32: "i", i64: "q", f32: "f", vp: "Q"}
    return "".join(codes.get(t) or _formats(t) for _, t in cls._fields_)


def packer(cls):
    """A function from the fields' values, in order, to the structure's bytes
    (pointers as addresses, 0 for NULL): a quarter of the time that filling
    the ctypes structure takes.  The entries that take it declare their
    argument ``c_void_p``, which reads a ``bytes`` object in place."""
    fmt = struct.Struct("@" + _formats(cls))
    if fmt.size != C.sizeof(cls):
        raise AssertionError(f"{cls.__name__}: packed {fmt.size} bytes, C {C.sizeof(cls)}")
    return fmt.pack


EXPORTS = {
    "hier_meta_count": [C.POINTER(HierTopo), C.POINTER(HierMetaCounts), vp],
    "hier_meta_build": [C.POINTER(HierTopo), C.POINTER(HierMetaOut), vp],
    "hier_derive_workspace": [C.POINTER(HierDeriveArgs)],
    "hier_derive_count": [C.POINTER(HierDeriveArgs), vp],
    "hier_derive_build": [C.POINTER(HierDeriveArgs), vp],
    "hier_derive_ste_classes": [C.POINTER(HierDeriveArgs), vp, vp, vp],
    "hier_membership_from_logits": [C.POINTER(HierMembershipArgs), vp],
    "hier_merge_hub_lists": [C.POINTER(HierMergeArgs), vp],
    "hier_trim_key_lists": [C.POINTER(HierTrimArgs), vp],
    "hier_trim_key_lists2": [C.POINTER(HierTrimArgs), C.POINTER(HierTrimArgs), vp],
    "hier_qkv_prologue": [C.POINTER(HierPrologueArgs), vp],
    "hier_qk_prologue_bwd_waves": [C.POINTER(HierPrologueBwdArgs)],
    "hier_qk_prologue_bwd": [C.POINTER(HierPrologueBwdArgs), vp],
    "hier_qk_prologue_grads": [C.POINTER(HierPrologueBwdArgs), C.POINTER(HierPrologueGradArgs), vp],
    "hier_attn_fwd": [C.POINTER(HierFwdArgs), vp],
    "hier_attn_bwd": [C.POINTER(HierBwdArgs), vp],
    "hier_attn_bwd_noalloc": [C.POINTER(HierBwdArgs), vp],
    "hier_ste_reduce": [C.POINTER(HierSteReduceArgs), vp],
    "hier_ste_logit_grad": [C.POINTER(HierSteReduceArgs), vp, vp],
    "hier_kv_append": [C.POINTER(HierPageArgs), vp],
    "hier_frame_attn": [C.POINTER(HierFrameAttnArgs), vp],
    "hier_gated_residual": [C.POINTER(HierGateArgs), vp],
    "hier_head_prologue": [vp, vp],
    "hier_head_prologue_bwd": [vp, vp],
    "hier_kv_append_fp8": [vp, vp],
    "hier_attn_fwd_fp8": [vp, vp],
    "hier_rms_norm": [vp, vp],
    "hier_rms_norm_bwd_rows": [vp],
    "hier_rms_norm_bwd": [vp, vp],
    "hier_linear_workspace": [vp],
    "hier_linear": [vp, vp],
    "hier_pad_rows": [vp, vp],
    "hier_linear_bwd_workspace": [vp],
    "hier_linear_bwd": [vp, vp],
    "hier_cross_workspace": [vp],
    "hier_cross_attn": [vp, vp],
    "hier_cross_bwd_workspace": [vp],
    "hier_cross_attn_bwd": [vp, vp],
    "hier_last_error": [],
    "hier_version": [],
}

_SIZES = ("hier_derive_workspace", "hier_rms_norm_bwd_rows", "hier_linear_workspace",
          "hier_linear_bwd_workspace", "hier_cross_workspace", "hier_cross_bwd_workspace")        # entries that return a size

_lock = threading.Lock()
_lib = None


def lib() -> C.CDLL:
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"hierattn HIP library not built: {LIB_PATH} is missing "
                    "(run `python -m multics_amd.build` or __graft_entry__.build())")
            handle = C.CDLL(str(LIB_PATH))
            for name, argtypes in EXPORTS.items():
                fn = getattr(handle, name)
                fn.argtypes = argtypes
                fn.restype = C.c_char_p if name in ("hier_last_error", "hier_version") else \
                    (C.c_int64 if name in _SIZES else C.c_int)
            _lib = handle
    return _lib


def check(rc: int, what: str) -> None:
    if rc == HIER_OK:
        return
    msg = f"{what}: {lib().hier_last_error().decode(errors='replace')}"
    if rc == HIER_EINVAL:
        raise ValueError(msg)
    if rc == HIER_EUNSUPPORTED:
        raise NotImplementedError(msg)
    if rc == HIER_EINTERNAL:
        raise AssertionError(msg)
    raise RuntimeError(msg)


def stream_of(device: torch.device) -> int:
    """The handle of PyTorch's current stream on ``device``, a GPU's (a launch
    handed host pointers would fault it): the number that
    ``torch.cuda.current_stream(device).cuda_stream`` gives, without the
    stream object."""
    if device.type != "cuda":
        raise ValueError(f"expected a GPU, got device {device}")
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args), name)


_functions = {}


def call_on(device: torch.device, name: str, *args) -> None:
    """``call`` with the current stream of ``device`` as the last argument,
    launched with that device current (a stream belongs to its device)."""
    if device.type != "cuda":
        raise ValueError(f"expected a GPU, got device {device}")
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(lib(), name)
    index, now = device.index, torch.cuda.current_device()
    if index is None or index == now:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(now))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous from a 16-byte address, copied if it is not."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def head_strides(t: torch.Tensor) -> tuple:
    """``t`` [S, H, D] readable in 16-byte rows (copied if it is not), and its
    strides over tokens and heads (0 where there is one only)."""
    for _ in range(2):
        ss, sh, unit = t.stride()
        ss, sh = ss if t.shape[0] > 1 else 0, sh if t.shape[1] > 1 else 0
        if unit == 1 and ss % 8 == 0 and sh % 8 == 0 and t.data_ptr() % 16 == 0:
            break
        t = aligned(t)
    return t, ss, sh
