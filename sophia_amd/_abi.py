"""The C ABI of ``libsophia_kda.so`` as a ctypes table, with no torch import.

Status codes, element types and flag bits of include/sophia_kda.h and every
entry point of include/sophia_kda.h, include/sophia_decoder.h,
include/sophia_draft.h and include/sophia_pages.h with its ctypes signature.  ``sophia_amd._native`` binds the library through this
table; the CPU tests also bind a host-sanitized build of the library with it
(torch is not loaded into that process).
"""

from __future__ import annotations

import ctypes

SOPHIA_OK = 0
SOPHIA_ERR_INVALID = 1
SOPHIA_ERR_HIP = 2
SOPHIA_ERR_WORKSPACE = 3

DTYPE_F32 = 0
DTYPE_BF16 = 1

QK_L2NORM = 1
GATE_IN_KERNEL = 2
BETA_SIGMOID = 4
SCAN_NO_SEGMENTS = 8
BWD_RECURRENT = 16
BWD_GRAD_BF16 = 32

TREE_NODES = 64          # SOPHIA_TREE_NODES of include/sophia_draft.h
BEAMS = 64               # SOPHIA_BEAMS, SOPHIA_MOVES, SOPHIA_FORK_MLA of include/sophia_pages.h
MOVES = 4096
POOLS = 24


class CommitKda(ctypes.Structure):
    """sophia_commit_kda of include/sophia_draft.h."""
    _fields_ = [("tape", ctypes.c_void_p), ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64),
                ("conv_state", ctypes.c_void_p), ("state", ctypes.c_void_p)]


class CommitMla(ctypes.Structure):
    """sophia_commit_mla of include/sophia_draft.h."""
    _fields_ = [("latent", ctypes.c_void_p), ("latent_stride", ctypes.c_int64), ("cache", ctypes.c_void_p),
                ("slot_stride", ctypes.c_int64)]


def packed(struct, words: list[int]):
    """An array of ``struct``, whose fields are 8 bytes each, from all its fields in a row (None: of
    nothing); field by field it would be a Python object for each."""
    if not words:
        return None
    flat = (ctypes.c_int64 * len(words))(*words)
    return (struct * (ctypes.sizeof(flat) // ctypes.sizeof(struct))).from_buffer(flat)


# Every symbol of include/sophia_kda.h, include/sophia_decoder.h,
# include/sophia_draft.h and include/sophia_pages.h, with its ctypes signature.
_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int
_f32 = ctypes.c_float
_u32 = ctypes.c_uint
_sz = ctypes.c_size_t
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "sophia_last_error": (ctypes.c_char_p, []),
    "sophia_abi_version": (_i32, []),
    "sophia_short_conv_fwd": (_i32, [_vp, _i64, _vp, _i64, _i32, _vp, _vp, _i32, _vp, _vp, _i32,
                                     _i64, _i32, _i32, _i32, _i32, _vp]),
    "sophia_short_conv_step": (_i32, [_vp, _i64, _vp, _i64, _i32, _vp, _vp, _i32, _vp, _i32, _i32,
                                      _i32, _i32, _vp]),
    "sophia_short_conv_bwd_workspace_size": (_sz, [_i64, _i32, _i32]),
    "sophia_short_conv_bwd": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _i32, _vp, _vp, _i32, _vp, _vp,
                                     _i32, _i64, _i32, _i32, _i32, _vp, _vp, _sz, _vp]),
    "sophia_kda_chunk_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "sophia_kda_chunk_fwd": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _i64, _i32,
                                    _vp, _vp, _f32, _f32, _u32, _vp, _vp, _i32, _i64, _i32, _i32,
                                    _vp, _vp, _i32, _vp, _vp, _i64, _vp, _sz, _vp]),
    "sophia_kda_chunk_fwd_no_alloc": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _i64,
                                             _i32, _vp, _vp, _f32, _f32, _u32, _vp, _vp, _i32, _i64,
                                             _i32, _i32, _vp, _vp, _i32, _vp, _vp, _i64, _vp]),
    "sophia_kda_decode_step": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _i64, _i32,
                                      _vp, _vp, _f32, _f32, _u32, _vp, _i32, _vp, _i32, _i32, _i32,
                                      _i32, _vp, _i64, _vp]),
    "sophia_kda_decode_conv_step": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _vp, _i32, _vp, _i64, _i32,
                                           _vp, _i64, _i32, _vp, _vp, _f32, _f32, _u32, _vp, _i32,
                                           _vp, _i32, _i32, _i32, _i32, _vp, _i64, _vp]),
    "sophia_kda_decode_mixer_step": (_i32, [_vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp,
                                            _f32, _f32, _u32, _vp, _i32, _vp, _i32, _vp, _i64, _vp, _f32, _i32, _i32,
                                            _i32, _vp, _i64, _vp]),
    "sophia_kda_conv_chunk_fwd": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _vp, _i32, _i32, _vp, _i64, _i32,
                                         _vp, _i64, _i32, _vp, _vp, _f32, _f32, _u32, _vp, _vp, _i32,
                                         _i64, _i32, _i32, _vp, _vp, _i32, _vp, _vp, _i64, _vp, _sz, _vp]),
    "sophia_mla_latent_norms": (_i32, [_vp, _i64, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _f32, _vp, _f32,
                                       _vp, _i32, _i32, _i64, _vp, _i32, _vp, _vp, _vp, _vp, _vp]),
    "sophia_kda_chunk_bwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "sophia_kda_chunk_bwd": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _i64, _i32, _vp, _i64, _i32,
                                    _vp, _vp, _f32, _f32, _u32, _vp, _i32, _i64, _i32, _i32,
                                    _vp, _vp, _i64, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                                    _vp, _vp, _sz, _vp]),
    "sophia_attn_res_mix": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i32, _vp, _vp,
                                   _f32, _vp, _f32, _vp, _i64, _i64, _i32, _i32, _vp]),
    "sophia_situ_glu": (_i32, [_vp, _i64, _vp, _i64, _i64, _i32, _f32, _f32, _i32, _vp]),
    "sophia_gated_head_norm": (_i32, [_vp, _i64, _i32, _vp, _i64, _vp, _f32, _vp, _i64, _i64, _i32,
                                      _i32, _i32, _vp]),
    "sophia_gated_head_norm_bwd_workspace_size": (_sz, [_i64, _i32, _i32]),
    "sophia_gated_head_norm_bwd": (_i32, [_vp, _i64, _vp, _i64, _i32, _vp, _i64, _vp, _f32, _vp, _i64,
                                          _vp, _i64, _vp, _i64, _i32, _i32, _i32, _vp, _sz, _vp]),
    "sophia_join_columns": (_i32, [_vp, _vp, _vp, _i32, _vp, _i64, _vp]),
    "sophia_row_linear": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp]),
    "sophia_row_linear_situ_glu": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _f32, _f32, _vp]),
    "sophia_head_linear": (_i32, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i32,
                                  _vp]),
    "sophia_head_linear_kn": (_i32, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _vp]),
    "sophia_mla_decode_workspace_size": (_sz, [_i64, _i32, _i32]),
    "sophia_causal_attention": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i32,
                                       _i64, _i64, _i32, _i32, _i32, _f32, _i32, _vp]),
    "sophia_mla_decode_attn": (_i32, [_vp, _i64, _i32, _vp, _i64, _i32, _i32, _vp, _vp, _f32, _vp,
                                      _i64, _i32, _i64, _i32, _i32, _i32, _vp, _sz, _vp]),
    "sophia_kda_tree_step": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _vp, _i32, _vp, _i64, _i32, _vp, _i64, _i32,
                                    _vp, _vp, _f32, _f32, _u32, _vp, _i32, _vp, _vp, _vp, _i32, _i64, _i32, _i32,
                                    _i32, _vp, _i64, _vp, _vp]),
    "sophia_tree_commit": (_i32, [_vp, _i64, _vp, _i32, _vp, _i32, _i64, _vp, _i32, _vp, _i32, _i32, _i32, _i32,
                                  _i32, _vp, _i32, _vp, _i32, _i32, _i32, _vp]),
    "sophia_tree_commit_within": (_i32, [_vp, _i64, _vp, _i32, _vp, _i32, _i64, _i32, _vp, _i32, _vp, _i32, _i32, _i32,
                                         _i32, _i32, _vp, _i32, _vp, _i32, _i32, _i32, _vp]),
    "sophia_mla_tree_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32]),
    "sophia_mla_tree_attn": (_i32, [_vp, _i64, _vp, _i64, _i32, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _i32,
                                    _i64, _i32, _f32, _vp, _i64, _i32, _i32, _i32, _i32, _vp, _sz, _vp]),
    "sophia_adjust_logits": (_i32, [_vp, _i64, _vp, _i64, _i32, _i64, _i32, _vp, _i64, _vp, _vp, _i32, _vp, _vp,
                                    _vp, _vp, _vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _i32, _i32, _vp]),
    "sophia_tree_accept_workspace_size": (_sz, [_i64, _i32]),
    "sophia_tree_accept": (_i32, [_vp, _i64, _i32, _i64, _i32, _vp, _vp, _vp, _i32, _i32, _vp, _i64, _vp, _vp, _vp,
                                  _vp, _sz, _vp]),
    "sophia_mla_paged_workspace_size": (_sz, [_i32, _i64, _i32, _i64, _i32, _i32, _i32, _i32]),
    "sophia_mla_paged_attn": (_i32, [_vp, _i64, _i32, _vp, _i64, _i64, _i32, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _i32,
                                     _i64, _i32, _i64, _f32, _vp, _i64, _i32, _i32, _i32, _vp, _sz, _vp]),
    "sophia_mla_latent_norms_paged": (_i32, [_vp, _i64, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _f32, _vp, _f32, _vp, _i64,
                                             _i64, _i32, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _i32, _vp]),
    "sophia_beam_select_workspace_size": (_sz, [_i64, _i32, _i32]),
    "sophia_beam_select": (_i32, [_vp, _i64, _i32, _i64, _i32, _vp, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _sz, _vp]),
    "sophia_move_workspace_size": (_sz, [_i32]),
    "sophia_cache_fork": (_i32, [_vp, _vp, _vp, _i32, _i32, _vp, _i64, _vp, _i64, _i32, _vp, _i64, _i32, _i32, _vp, _i64,
                                 _i64, _i32, _i32, _vp, _i64, _i32, _i32, _i32, _vp, _sz, _vp]),
    "sophia_page_copy": (_i32, [_vp, _vp, _i32, _vp, _i32, _i64, _i64, _i64, _i32, _vp, _sz, _vp]),
    "sophia_tree_accept_strict": (_i32, [_vp, _i64, _i32, _i64, _i32, _vp, _vp, _vp, _i32, _i32, _vp, _i64, _vp, _vp, _vp,
                                         _vp, _sz, _vp]),
}



def bind(path: str, mode: int = ctypes.DEFAULT_MODE) -> ctypes.CDLL:
    """Load the library at ``path`` and set every entry point's signature."""
    handle = ctypes.CDLL(path, mode=mode)
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return handle
