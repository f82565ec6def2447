"""ctypes declarations of the C ABI in include/mfmoe.h.

Loads the in-tree libmfmoe.so and fails loudly when it is missing: there is no
CPU fallback for any operator.
"""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmfmoe.so")

GROUP_SIZE = 64
MAX_TOKENS = 8
MAX_TOPK = 8
MAX_EXPERTS = 512
STATIC_ACT_ELEMS = MAX_TOKENS * 32768  # MF_STATIC_ACT_ELEMS

BITS_TERNARY, BITS_2, BITS_4, BITS_8 = 1, 2, 4, 8
ROUTER_TOPK_SOFTMAX, ROUTER_FULL_SOFTMAX = 0, 1

MAX_ROWS = 1 << 20         # MF_MAX_ROWS
MAX_ADAPTERS = 1024        # MF_MAX_ADAPTERS
MAX_ADAPTER_RANK = 256     # MF_MAX_ADAPTER_RANK
MAX_ADAPTER_TARGETS = 4    # MF_MAX_ADAPTER_TARGETS
GATE_NONE, GATE_ROW, GATE_ELEMENT, GATE_CHANNEL = 0, 1, 2, 3
ACT_NONE, ACT_SILU, ACT_GELU_TANH, ACT_GELU = 0, 1, 2, 3
BF16_EXPERTS_ROWS = 64     # MF_BF16_EXPERTS_ROWS
SAME_POSITIONS = 0xFFFFFFFF  # MF_SAME_POSITIONS

STATUS_NAMES = {
    0: "MF_OK", -1: "MF_ERR_INVALID_ARGUMENT", -2: "MF_ERR_DIMENSION_MISMATCH",
    -3: "MF_ERR_UNSUPPORTED_BITS", -4: "MF_ERR_SCRATCH_TOO_SMALL", -5: "MF_ERR_NO_DEVICE",
    -6: "MF_ERR_OUT_OF_MEMORY", -7: "MF_ERR_LAUNCH", -10: "MF_ERR_QUERY_COUNT",
    -11: "MF_ERR_TOPK", -12: "MF_ERR_NUM_EXPERTS", -13: "MF_ERR_TILE_EXPERT_COUNT",
    -14: "MF_ERR_PAIR_COUNT", -15: "MF_ERR_TOKEN_RANGE", -16: "MF_ERR_RANK_RANGE",
    -17: "MF_ERR_EXPERT_RANGE", -18: "MF_ERR_DUPLICATE_TOKEN_RANK", -19: "MF_ERR_SORT_KEY_COUNT",
}


class ExpertOffsets(C.Structure):
    """mf_expert_offsets (MoEExpertOffsets, Kernels/MoE/MoE.swift:4-29)."""
    _fields_ = [(n, C.c_uint32) for n in (
        "gate_w", "gate_s", "gate_b", "up_w", "up_s", "up_b", "down_w", "down_s", "down_b")]


class QTensor(C.Structure):
    """mf_qtensor: device pointers of one quantized projection."""
    _fields_ = [("weights", C.c_void_p), ("scales", C.c_void_p), ("biases", C.c_void_p)]


class MoEConfig(C.Structure):
    _fields_ = [
        ("d", C.c_uint32), ("f", C.c_uint32), ("num_experts", C.c_uint32), ("top_k", C.c_uint32),
        ("bits", C.c_int), ("router_mode", C.c_int), ("swiglu_limit", C.c_float),
        ("shared_f", C.c_uint32), ("shared_bits", C.c_int), ("maple_rounding", C.c_uint32),
        ("gate_group_size", C.c_uint32),
    ]


class LayerWeights(C.Structure):
    _fields_ = [
        ("router_w", C.c_void_p), ("expert_base", C.c_void_p), ("expert_stride", C.c_size_t),
        ("offsets", ExpertOffsets),
        ("shared_gate", QTensor), ("shared_up", QTensor), ("shared_down", QTensor),
        ("w_sg", C.c_void_p),
        ("w_sg_q8", QTensor),
        ("expert_tiled", C.c_void_p),
    ]


class Pair(C.Structure):
    _fields_ = [("token", C.c_uint32), ("expert", C.c_uint32), ("rank", C.c_uint32),
                ("weight_bits", C.c_uint32)]


class AdapterPool(C.Structure):
    """mf_adapter_pool"""
    _fields_ = [("num_adapters", C.c_uint32), ("rank", C.c_uint32), ("n", C.c_uint32),
                ("ranks", C.c_void_p), ("scales", C.c_void_p)]


class AdapterTarget(C.Structure):
    """mf_adapter_target"""
    _fields_ = [("a", C.c_void_p), ("b", C.c_void_p), ("y", C.c_void_p), ("m", C.c_uint32), ("y_stride", C.c_uint32)]


class BlockNormArgs(C.Structure):
    """mf_block_norm_args"""
    _fields_ = [("hidden", C.c_void_p), ("delta", C.c_void_p), ("gate", C.c_void_p), ("post_weight", C.c_void_p),
                ("pre_weight", C.c_void_p), ("out", C.c_void_p), ("d", C.c_uint32), ("t", C.c_uint32),
                ("hidden_stride", C.c_uint32), ("delta_stride", C.c_uint32), ("gate_stride", C.c_uint32), ("out_stride", C.c_uint32),
                ("delta_f32", C.c_int), ("gate_kind", C.c_int), ("post_eps", C.c_float), ("pre_eps", C.c_float),
                ("residual_scale", C.c_float), ("branch_scale", C.c_float), ("weight_bias", C.c_float)]


class ProjectArgs(C.Structure):
    """mf_project_args"""
    _fields_ = [("x", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p), ("y", C.c_void_p),
                ("t", C.c_uint32), ("m", C.c_uint32), ("n", C.c_uint32),
                ("x_stride", C.c_uint32), ("w_stride", C.c_uint32), ("residual_stride", C.c_uint32), ("y_stride", C.c_uint32),
                ("y_f32", C.c_int), ("gated", C.c_int), ("activation", C.c_int)]


class HeadRows(C.Structure):
    """mf_head_rows"""
    _fields_ = [("x", C.c_void_p), ("out", C.c_void_p), ("weight", C.c_void_p), ("heads", C.c_uint32),
                ("row_stride", C.c_uint32), ("head_stride", C.c_uint32), ("out_row_stride", C.c_uint32), ("out_head_stride", C.c_uint32)]


class HeadNormsArgs(C.Structure):
    """mf_head_norms_args"""
    _fields_ = [("q", HeadRows), ("k", HeadRows), ("positions", C.c_void_p), ("inv_freq", C.c_void_p), ("axis_of_pair", C.c_void_p),
                ("t", C.c_uint32), ("head_dim", C.c_uint32), ("rotary_dim", C.c_uint32), ("axes", C.c_uint32), ("position_stride", C.c_uint32),
                ("interleaved", C.c_int), ("eps", C.c_float), ("weight_bias", C.c_float), ("rotation_scale", C.c_float)]


class Bf16ExpertPool(C.Structure):
    """mf_bf16_expert_pool"""
    _fields_ = [(n, C.c_void_p) for n in ("gate_up", "down", "gate_up_bias", "down_bias", "shared_gate_up", "shared_down", "shared_gate")] + [
        (n, C.c_uint32) for n in ("num_experts", "top_k", "d", "f", "shared_f")] + [("activation", C.c_int)]


# every entry point include/mfmoe.h declares: name -> (restype, argtypes)
_P, _SZ, _U32, _I = C.c_void_p, C.c_size_t, C.c_uint32, C.c_int
SIGNATURES = {
    "mf_abi_version": (_I, []),
    "mf_status_string": (C.c_char_p, [_I]),
    "mf_ctx_create": (_I, [_I, C.POINTER(_P)]),
    "mf_ctx_destroy": (None, [_P]),
    "mf_last_hip_error": (C.c_char_p, [_P]),
    "mf_quantize_affine": (_I, [_P, _P, _P, _SZ, _SZ, _I, _P, _P, _P]),
    "mf_dequantize": (_I, [_P, _P, QTensor, _SZ, _SZ, _I, _P]),
    "mf_gemv": (_I, [_P, _P, QTensor, _I, _P, _P, _U32, _U32, _U32, _I]),
    "mf_silu_mul": (_I, [_P, _P, _P, _P, _P, _U32]),
    "mf_sigmoid_scalar_mul": (_I, [_P, _P, _P, _P, _U32, _U32]),
    "mf_residual_add": (_I, [_P, _P, _P, _P, _U32]),
    "mf_residual_rmsnorm": (_I, [_P, _P, _P, _P, _P, _P, _U32, _U32, C.c_float]),
    "mf_shared_expert": (_I, [_P, _P, _P, QTensor, QTensor, QTensor, _I, _U32, _U32, _U32, _P, _P,
                              _SZ]),
    "mf_shared_expert_scratch_bytes": (_SZ, [_U32, _U32, _U32]),
    "mf_shared_expert_int8": (_I, [_P, _P, _P, QTensor, QTensor, QTensor, _U32, _U32, _U32, _I, _P, _P, _SZ]),
    "mf_qmm_workspace_bytes": (_SZ, [_U32, _U32, _U32]),
    "mf_qmm": (_I, [_P, _P, QTensor, _I, _P, _P, _U32, _U32, _U32, _I, _P, _SZ]),
    "mf_qmm_path": (_I, [QTensor, _I, _P, _P, _U32, _U32, _U32, _P, _SZ]),
    "mf_shared_expert_static": (_I, [_P, _P, _P, QTensor, QTensor, QTensor, _I, _U32, _U32, _U32, _P]),
    "mf_expert_blob_layout": (_I, [_U32, _U32, _I, _U32, C.POINTER(ExpertOffsets), C.POINTER(_SZ), C.POINTER(_SZ)]),
    "mf_expert_blob_layout_repacked": (_I, [_U32, _U32, _I, _U32, C.POINTER(ExpertOffsets), C.POINTER(_SZ), C.POINTER(_SZ)]),
    "mf_moe_config_check": (_I, [C.POINTER(MoEConfig)]),
    "mf_moe_create": (_I, [_P, C.POINTER(MoEConfig), C.POINTER(_P)]),
    "mf_moe_destroy": (None, [_P]),
    "mf_moe_router": (_I, [_P, _P, _P, _P, _U32, _U32, _P, _P, _P]),
    "mf_router_sqrtsoftplus": (_I, [_P, _P, _P, _P, _U32, _U32, _U32, _U32, _U32, _P, C.c_float, _P, _P, _P]),
    "mf_router_hash_weights": (_I, [_P, _P, _P, _P, _U32, _U32, _U32, _U32, _U32, _P, C.c_float, _P, _P]),
    "mf_router_inkling": (_I, [_P, _P, _P, _P, _U32, _U32, _U32, _U32, _U32, _U32, _P, _P, C.c_float, _P,
                               _P, _P, _P]),
    "mf_router_gemma4": (_I, [_P, _P, _P, _P, _P, _P, _U32, _U32, _P, _P, _U32, _U32, _U32, _P, _P, _P]),
    "mf_moe_phase1": (_I, [_P, _P, _P, _SZ, C.POINTER(ExpertOffsets), _P, _P, _U32, _U32, _P]),
    "mf_moe_phase1_subset": (_I, [_P, _P, _P, _SZ, C.POINTER(ExpertOffsets), _P, _P, _U32, _U32, _P, _P, _U32]),
    "mf_moe_phase2": (_I, [_P, _P, _P, _SZ, C.POINTER(ExpertOffsets), _P, _P, _P, _P, _U32, _P]),
    "mf_moe_decode_layer": (_I, [_P, _P, C.POINTER(LayerWeights), _P, _U32, _P, _P, _P, _P]),
    "mf_moe_decode_layer_normed": (_I, [_P, _P, C.POINTER(LayerWeights), _P, _P, _P, C.c_float, _U32, _P, _P, _P]),
    "mf_moe_set_fused": (_I, [_P, _I]),
    "mf_moe_set_prefill_route_rounding": (_I, [_P, _I]),
    "mf_moe_tile_experts": (_I, [_P, _P, _P, _SZ, C.POINTER(ExpertOffsets), _P]),
    "mf_moe_status": (_I, [_P, _P]),
    "mf_moe_set_phase_trace": (_I, [_P, _P, _SZ]),
    "mf_ctx_num_cu": (_I, [_P]),
    "mf_moe_group": (_I, [_P, _P, _P, _P, _U32, _P, _P, _P]),
    "mf_moe_group_status": (_I, [_P, _P]),
    "mf_moe_prefill_workspace_bytes": (_SZ, [_P, _U32]),
    "mf_moe_prefill_layer": (_I, [_P, _P, C.POINTER(LayerWeights), _P, _U32, _P, _P, _SZ, _P, _P]),
    "mf_moe_slot_lookup": (_I, [_P, _P, _P, _U32, _P, C.c_uint64, _P, _P]),
    "mf_moe_phase1_slots": (_I, [_P, _P, _P, _P, _P, C.POINTER(ExpertOffsets), _P, _U32, _U32, _P]),
    "mf_moe_phase2_slots": (_I, [_P, _P, _P, _P, _P, C.POINTER(ExpertOffsets), _P, _P, _P, _U32, _P]),
    "mf_moe_ragged_qmm": (_I, [_P, _P, _P, _SZ, C.POINTER(ExpertOffsets), _P, _P, _P, _U32, _P, _P, _SZ]),
    "mf_moe_unpermute": (_I, [_P, _P, _P, _P, _P, _P, _U32, _P]),
    "mf_adapter_plan_bytes": (_SZ, [_U32, _U32]),
    "mf_adapter_group": (_I, [_P, _P, _P, _U32, _U32, _P, _SZ]),
    "mf_adapter_workspace_bytes": (_SZ, [C.POINTER(AdapterPool), _U32, _U32]),
    "mf_adapter_apply": (_I, [_P, _P, C.POINTER(AdapterPool), _P, _U32, _P, _U32, _P, _U32, _I, _P, _P, _SZ]),
    "mf_block_norm": (_I, [_P, _P, _P]),
    "mf_project_workspace_bytes": (_SZ, [_U32, _U32, _U32, _I]),
    "mf_project": (_I, [_P, _P, _P, _P, _SZ]),
    "mf_head_norms": (_I, [_P, _P, _P]),
    "mf_bf16_experts_workspace_bytes": (_SZ, [C.POINTER(Bf16ExpertPool), _U32]),
    "mf_bf16_experts": (_I, [_P, _P, C.POINTER(Bf16ExpertPool), _P, _U32, _P, _P, _P, _U32, _U32, _P, _U32, _P, _SZ]),
    "mf_group_pairs_host": (_I, [_P, _SZ, _I, _I, _I, _I, _P, _SZ, _P, _P, _P, _P,
                                 C.POINTER(_SZ), _P, C.POINTER(_SZ), _P]),
}

_lib = None


class LibraryMissing(RuntimeError):
    pass


def lib() -> C.CDLL:
    """The loaded libmfmoe.so.  Raises LibraryMissing if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise LibraryMissing(
                f"{LIB_PATH} is missing: build it with `python -m mference_amd.build` "
                "(there is no CPU fallback)")
        # torch carries its own HIP runtime; it has to be the one already loaded
        # when libmfmoe resolves libamdhip64, or device pointers and streams
        # would belong to a different runtime instance than the kernels.
        import torch  # noqa: F401
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


class MfError(RuntimeError):
    """A negative mf_status (the reference's `throws` / precondition failures)."""

    def __init__(self, status: int, detail: str = ""):
        self.status = status
        self.name = STATUS_NAMES.get(status, str(status))
        text = lib().mf_status_string(status).decode()
        super().__init__(f"{self.name}: {text}" + (f" ({detail})" if detail else ""))


def check(status: int, ctx=None) -> None:
    if status != 0:
        detail = ""
        if status == -7 and ctx:
            detail = lib().mf_last_hip_error(ctx).decode()
        raise MfError(status, detail)
