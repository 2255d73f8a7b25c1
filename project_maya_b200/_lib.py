"""Loader of the C-ABI library (libmaya_moe.so) and its ctypes signatures.

There is no fallback: if the library has not been built, importing the compute entry points raises.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

PKG = Path(__file__).resolve().parent
# MAYA_MOE_LIB: another build of the same library (comparing two builds on one machine); it must export the same ABI
LIB_PATH = Path(os.environ.get("MAYA_MOE_LIB") or PKG / "libmaya_moe.so")

c_void_p, c_int, c_float, c_size_t, c_int64, c_uint64 = C.c_void_p, C.c_int, C.c_float, C.c_size_t, C.c_int64, C.c_uint64


class ExpertLayout(C.Structure):
    _fields_ = [("gu_type", c_int), ("d_type", c_int), ("n_embd", c_int64), ("n_ff", c_int64),
                ("gu_row", c_size_t), ("d_row", c_size_t), ("up_off", c_size_t), ("down_off", c_size_t),
                ("bytes", c_size_t), ("u_type", c_int), ("u_row", c_size_t)]


class MoePlan(C.Structure):
    _fields_ = [("plan_ptr", c_void_p), ("plan_w", c_void_p), ("cpu_part", c_void_p), ("cpu_flag", c_void_p),
                ("skip", c_void_p)]


class MoeWin(C.Structure):
    _fields_ = [("plan_ptr", c_void_p), ("plan_w", c_void_p), ("cpu_part", c_void_p), ("cpu_flag", c_void_p),
                ("xq", c_void_p), ("xq_stride", c_size_t), ("hq", c_void_p), ("part", c_void_p), ("sh_out", c_void_p),
                ("out", c_void_p), ("out_stride", c_size_t), ("grp_ptr", c_void_p), ("grp_start", c_void_p),
                ("grp_ent", c_void_p), ("n_groups", c_void_p), ("T", c_int), ("k", c_int), ("n_embd", c_int),
                ("n_ff", c_int), ("limit", c_float), ("down_off", c_size_t)]


class MoeLayerDesc(C.Structure):
    _fields_ = [("n_embd", c_int), ("n_ff", c_int), ("n_expert", c_int), ("k", c_int), ("gu_type", c_int),
                ("d_type", c_int), ("experts", c_void_p), ("expert_stride", c_size_t), ("n_ff_sh", c_int),
                ("sh_gu_type", c_int), ("sh_d_type", c_int), ("shared", c_void_p), ("limit", c_float),
                ("expert_lo", c_int), ("expert_hi", c_int), ("shared_here", c_int), ("staged", c_int), ("sh_lo", c_int),
                ("sh_hi", c_int), ("router", c_int), ("router_bias", c_void_p), ("router_w_scale", c_float),
                ("router_norm_w", c_int), ("cpu_part", c_void_p), ("cpu_flag", c_void_p)]


class MmqProduct(C.Structure):
    _fields_ = [("w", c_void_p), ("type", c_int), ("w_rows", c_int64), ("w_cols", c_int64), ("expert_bytes", c_size_t),
                ("n", c_int), ("xq", c_void_p), ("bounds", c_void_p), ("ids", c_void_p), ("total_rows", c_int64),
                ("max_rows", c_int64), ("dst", c_void_p), ("ld_dst", c_int64), ("expert_map", c_void_p),
                ("error", c_void_p), ("xq_out", c_void_p)]


class PeerArFailure(C.Structure):
    _fields_ = [("captured", C.c_uint), ("sequence", C.c_uint), ("observed", C.c_uint), ("block", C.c_uint),
                ("n4", C.c_uint), ("rank", C.c_uint), ("waited_for", C.c_uint), ("pad", C.c_uint),
                ("elapsed_ns", C.c_ulonglong), ("timeout_ns", C.c_ulonglong)]


class PeerArDesc(C.Structure):
    _fields_ = [("recv", c_void_p), ("peer_recv", c_void_p), ("flags", c_void_p), ("peer_flags", c_void_p),
                ("error", c_void_p), ("failure", c_void_p), ("stride", c_size_t), ("timeout_ns", C.c_ulonglong),
                ("nm", c_int), ("seq_counter", c_void_p)]


class HcPostArgs(C.Structure):
    _fields_ = [("R_old", c_void_p), ("post", c_void_p), ("comb", c_void_p), ("R_new", c_void_p)]


class LoraArgs(C.Structure):
    _fields_ = [("x", c_void_p), ("y", c_void_p), ("out", c_void_p), ("a", c_void_p), ("b", c_void_p), ("scale", c_void_p), ("idx", c_void_p),
                ("scratch", c_void_p), ("scratch_bytes", c_size_t), ("ld_x", c_int64), ("ld_y", c_int64), ("ld_out", c_int64), ("n_tokens", c_int),
                ("n_in", c_int), ("n_out", c_int), ("rank", c_int), ("n_adapters", c_int), ("x_is_bf16", c_int), ("w_is_f16", c_int), ("kernel", c_int)]


class RouteArgs(C.Structure):
    _fields_ = [("logits", c_void_p), ("bias", c_void_p), ("n_tokens", c_int), ("n_expert", c_int), ("k", c_int), ("n_group", c_int),
                ("n_keep", c_int), ("sigmoid", c_int), ("top2", c_int), ("norm_w", c_int), ("w_scale", c_float), ("ids", c_void_p),
                ("weights", c_void_p)]


class RmsArgs(C.Structure):
    _fields_ = [("h", c_void_p), ("add", c_void_p), ("w", c_void_p), ("h_out", c_void_p), ("x_out", c_void_p), ("xq", c_void_p),
                ("ld_h", c_int64), ("ld_add", c_int64), ("ld_h_out", c_int64), ("ld_x", c_int64), ("n_rows", c_int64), ("n", c_int),
                ("eps", c_float), ("h_is_bf16", c_int), ("add_is_bf16", c_int), ("x_is_bf16", c_int), ("image", c_int)]


class KvCacheDesc(C.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p), ("k_sum", c_void_p),
                ("table", c_void_p), ("table_ld", c_int), ("n_blocks", c_int), ("n_kv", c_int), ("head_dim", c_int)]


class AttnBatchDesc(C.Structure):
    _fields_ = [("start", c_void_p), ("kv_len", c_void_p), ("n_seq", c_int), ("n_tokens", c_int), ("max_new", c_int), ("max_len", c_int)]


class KvPagesDesc(C.Structure):
    _fields_ = [("layers", c_void_p), ("table", c_void_p), ("refs", c_void_p), ("scratch", c_void_p), ("scratch_bytes", c_size_t),
                ("n_seq", c_int), ("table_ld", c_int), ("n_blocks", c_int), ("n_layers", c_int), ("n_kv", c_int), ("head_dim", c_int),
                ("has_sums", c_int)]


class RopeArgs(C.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("ld_q", c_int64), ("ld_k", c_int64), ("ld_v", c_int64),
                ("is_bf16", c_int), ("n_q", c_int), ("q_w", c_void_p), ("k_w", c_void_p), ("eps", c_float), ("cos", c_void_p),
                ("sin", c_void_p), ("pos", c_void_p), ("n_pos", c_int), ("rot_dim", c_int), ("pairs", c_int), ("q_out", c_void_p)]


class AttnArgs(C.Structure):
    _fields_ = [("q", c_void_p), ("ld_q", c_int64), ("is_bf16", c_int), ("n_q", c_int), ("scale", c_float), ("window", c_int),
                ("sel", c_void_p), ("n_sel", c_int), ("out", c_void_p), ("lse", c_void_p)]


class SelectArgs(C.Structure):
    _fields_ = [("q", c_void_p), ("ld_q", c_int64), ("is_bf16", c_int), ("n_q", c_int), ("n_first", c_int), ("n_last", c_int),
                ("n_sel", c_int), ("sel", c_void_p)]


_SIGNATURES = {
    "maya_version": (C.c_char_p, []),
    "maya_last_cuda_error": (c_int, []),
    "maya_launch_errors": (c_int, []),
    "maya_launch_count": (C.c_longlong, []),
    "maya_device_ok": (c_int, []),
    "maya_type_supported": (c_int, [c_int]),
    "maya_row_bytes": (c_size_t, [c_int, c_int64]),
    "maya_weight_bytes": (c_size_t, [c_int, c_int, c_int]),
    "maya_q8_1_bytes": (c_size_t, [c_int, c_int]),
    "maya_expert_layout_make": (c_int, [c_int, c_int, c_int, c_int64, c_int64, C.POINTER(ExpertLayout)]),
    "maya_router_top10": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "maya_router_sigmoid": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_float, c_int, c_void_p, c_void_p, c_void_p]),
    "maya_quantize_q8_1": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p]),
    "maya_quantize_q8_1_bf16": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p]),
    "maya_swiglu_q8_1": (c_int, [c_void_p, c_void_p, c_float, c_int64, c_void_p, c_void_p]),
    "maya_mmvq": (c_int, [c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "maya_moe_gate_up": (c_int, [c_int, C.POINTER(MoePlan), c_int, c_int, c_int, c_float, c_void_p, c_void_p, c_void_p,
                                 c_int, c_void_p, c_int, c_void_p, c_void_p]),
    "maya_moe_down": (c_int, [c_int, C.POINTER(MoePlan), c_int, c_int, c_int, c_size_t, c_void_p, c_void_p, c_void_p,
                              c_void_p]),
    "maya_moe_win_experts": (c_int, [c_int, c_int, C.POINTER(MoeWin), c_void_p]),
    "maya_moe_win_experts_checked": (c_int, [c_int, c_int, C.POINTER(MoeWin), C.c_uint, c_void_p, c_void_p]),
    "maya_moe_win_group": (c_int, [C.POINTER(MoeWin), c_void_p]),
    "maya_expert_scratch_bytes": (c_size_t, [c_int64, c_int64]),
    "maya_expert_grouped": (c_int, [C.POINTER(ExpertLayout), c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                    c_int64, c_void_p, c_void_p, c_void_p, c_void_p, c_float]),
    "maya_expert_static_scratch_bytes": (c_size_t, []),
    "maya_expert_grouped_static": (c_int, [C.POINTER(ExpertLayout), c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                           c_int64, c_void_p, c_void_p, c_void_p, c_float]),
    "maya_moe_combine": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "maya_expert_count": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "maya_expert_bounds": (c_int, [c_void_p, c_int, c_void_p, c_void_p]),
    "maya_expert_group_counts": (c_int, [c_void_p, c_int, c_int, c_int, *[c_void_p] * 6]),
    "maya_expert_group": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "maya_expert_scatter": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "maya_swiglu_rows": (c_int, [c_void_p, c_void_p, c_int, c_int, c_float, c_int, c_void_p]),
    "maya_moe_combine_rows": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p]),
    "maya_rms_router": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p,
                                c_void_p]),
    "maya_router_groups": (c_int, [C.POINTER(RouteArgs), c_void_p]),
    "maya_moe_layer_decode_routed": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
    "maya_pages_scratch_bytes": (c_size_t, [C.POINTER(KvPagesDesc)]),
    "maya_pages_reserve": (c_int, [C.POINTER(KvPagesDesc), C.POINTER(AttnBatchDesc), c_void_p]),
    "maya_pages_fork": (c_int, [C.POINTER(KvPagesDesc), c_void_p, c_void_p, c_void_p, c_int, c_void_p]),
    "maya_pages_free": (c_int, [C.POINTER(KvPagesDesc), c_void_p, c_int, c_void_p]),
    "maya_pages_compact": (c_int, [C.POINTER(KvPagesDesc), c_int, c_void_p]),
    "maya_pages_copy": (c_int, [C.POINTER(KvPagesDesc), c_void_p, c_void_p, c_int, c_void_p]),
    "maya_pages_error": (c_int, [C.POINTER(KvPagesDesc), c_void_p]),
    "maya_lora_scratch_bytes": (c_size_t, [c_int, c_int, c_int, c_int]),
    "maya_lora_error": (c_int, [c_void_p, c_void_p]),
    "maya_lora": (c_int, [C.POINTER(LoraArgs), c_void_p]),
    "maya_rms_q8": (c_int, [C.POINTER(RmsArgs), c_void_p]),
    "maya_q8_read": (c_int, [c_void_p, c_int, c_int64, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "maya_mmq_supported": (c_int, [c_int]),
    "maya_mmq_q8_bytes": (c_size_t, [c_int64, c_int64]),
    "maya_mmq_quantize": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "maya_mmq_quantize_bf16": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "maya_mmq_quantize_routed": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "maya_mmq_quantize_routed_bf16": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "maya_mmq_run": (c_int, [C.POINTER(MmqProduct), c_void_p]),
    "maya_mmq_run_glu": (c_int, [C.POINTER(MmqProduct), c_float, c_void_p]),
    "maya_mmq_chain_bytes": (c_size_t, [c_int64, c_int, c_int]),
    "maya_mmq_run_chain": (c_int, [C.POINTER(MmqProduct), C.POINTER(MmqProduct), c_int, c_float, c_void_p, c_size_t, c_void_p]),
    "maya_moe_combine_rows_local": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_int, c_int, c_int,
                                            c_void_p, c_void_p]),
    "maya_moe_combine_rows_local_ar": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_int, c_int, c_int,
                                               c_void_p, c_void_p, c_int, C.c_uint, c_void_p]),
    "maya_moe_combine_add": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p]),
    "maya_moe_layer_scratch_bytes": (c_size_t, [C.POINTER(MoeLayerDesc), c_int]),
    "maya_moe_layer_error": (c_int, [C.POINTER(MoeLayerDesc), c_int, c_void_p, c_void_p]),
    "maya_moe_layer_phase_ns": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, C.POINTER(C.c_ulonglong)]),
    "maya_moe_layer_decode": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p,
                                      c_void_p, c_void_p, c_size_t, c_void_p]),
    "maya_moe_layer_kernel": (c_int, [C.POINTER(MoeLayerDesc), c_int, c_int]),
    "maya_moe_layer_decode_checked": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
                                              c_size_t, c_int, C.c_uint, C.POINTER(HcPostArgs), c_void_p]),
    "maya_peer_ar_recv_bytes": (c_size_t, [c_int, c_size_t]),
    "maya_peer_ar_flag_bytes": (c_size_t, [c_int]),
    "maya_peer_ar_preload": (c_int, [c_void_p]),
    "maya_allreduce_peer": (c_int, [c_void_p, c_int, C.POINTER(PeerArDesc), c_int, C.c_uint, c_void_p]),
    "maya_moe_layer_decode_ar": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p,
                                         c_void_p, c_void_p, c_size_t, C.POINTER(PeerArDesc), c_int, C.c_uint, c_void_p]),
    "maya_hc_post": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p]),
    "maya_moe_layer_decode_hc": (c_int, [C.POINTER(MoeLayerDesc), c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p,
                                         c_void_p, c_void_p, c_size_t, C.POINTER(PeerArDesc), c_int, C.c_uint,
                                         C.POINTER(HcPostArgs), c_void_p]),
    "maya_peer_buffer_create": (c_int, [c_size_t, C.POINTER(c_void_p), C.c_char_p]),
    "maya_peer_buffer_open": (c_int, [C.c_char_p, C.POINTER(c_void_p)]),
    "maya_peer_buffer_close": (c_int, [c_void_p]),
    "maya_peer_buffer_destroy": (c_int, [c_void_p]),
    "maya_quantize_weights_host": (c_int, [c_int, c_void_p, c_int64, c_int64, c_void_p]),
    "maya_qk_norm_rope_append": (c_int, [C.POINTER(KvCacheDesc), C.POINTER(AttnBatchDesc), C.POINTER(RopeArgs), c_void_p]),
    "maya_kv_read": (c_int, [C.POINTER(KvCacheDesc), c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p]),
    "maya_attn_scratch_bytes": (c_size_t, [C.POINTER(KvCacheDesc), c_int, c_int]),
    "maya_attn_q8": (c_int, [C.POINTER(KvCacheDesc), C.POINTER(AttnBatchDesc), C.POINTER(AttnArgs), c_void_p, c_size_t, c_void_p]),
    "maya_attn_error": (c_int, [c_void_p, c_void_p]),
    "maya_block_select": (c_int, [C.POINTER(KvCacheDesc), C.POINTER(AttnBatchDesc), C.POINTER(SelectArgs), c_void_p]),
    "maya_synth_weights": (c_int, [c_int, c_uint64, c_float, c_int64, c_int64, c_void_p, c_void_p]),
}

_lib = None


def load() -> C.CDLL:
    """The loaded library; raises if it has not been built (python -m project_maya_b200.build)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m project_maya_b200.build` "
                               "(there is no CPU or PyTorch fallback for this path)")
        lib = C.CDLL(str(LIB_PATH))
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def declared_symbols() -> list[str]:
    return sorted(_SIGNATURES)
