"""ctypes binding of the C-ABI in include/forge_amd.h (libforge_amd.so).

Loading fails loudly when the library has not been built: there is no CPU or
PyTorch fallback for any operator of this package.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libforge_amd.so")
BINDING_PATH = os.path.join(HERE, "lib", "forge_torch.so")

FORGE_OK = 0
FORGE_EINVAL = -1
FORGE_ENODEV = -2
FORGE_ERANGE = -3

_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
_F = ctypes.c_float

# name -> (restype, argtypes); mirrors include/forge_amd.h one to one.
SIGNATURES = {
    "forge_status_string": (ctypes.c_char_p, [_I]),
    "forge_init": (_I, []),
    "forge_ksplit_last": (_I, [_P, _P]),
    "forge_ksplit_reset": (_I, [_P]),
    "forge_slots_in_use": (_I, [_P, _P, _P, _P]),
    "forge_last_route": (ctypes.c_char_p, []),
    "forge_get_compute_capability": (_I, [_I, _P]),
    "forge_has_int8_matrix_cores": (_I, [_I, _P]),
    "forge_quantize_activation": (_I, [_P, _P, _P, _I, _I, _P]),
    "forge_quantize_activation_twopass": (_I, [_P, _P, _P, _I, _I, _I, _P]),
    "forge_dequantize_bias": (_I, [_P, _P, _P, _P, _P, _I, _I, _P]),
    "forge_int8_gemm_dequant": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P]),
    "forge_int8_gemm": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P]),
    "forge_int8_linear": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _P]),
    "forge_int8_gemm_s32": (_I, [_P, _P, _P, _I, _I, _I, _P]),
    "forge_int8_linear_backward_prep": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P]),
    "forge_int8_linear_noalloc": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _P]),
    "forge_prune_compress_24": (_I, [_P, _P, _P, _I, _I, _P]),
    "forge_pack_metadata": (_I, [_P, _P, _I, _I, _P]),
    "forge_unpack_metadata": (_I, [_P, _P, _I, _I, _P]),
    "forge_sparse_int8_gemm_plan": (_I, [_I, _I, _I, _I, _I, _I, _P, _P]),
    "forge_sparse_int8_gemm": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _I, _P, _I]),
    "forge_sparse_int8_gemm_s32": (_I, [_P, _P, _P, _P, _I, _I, _I, _P]),
    "forge_sparse_int8_linear_fused": (_I, [_I, _I, _I, _P]),
    "forge_sparse_int8_linear": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _P, _I, _P, _I]),
    "forge_splitk_reduce": (_I, [_P, _P, _P, _I, _I, _P]),
    "forge_int8_conv2d_workspace_size": (ctypes.c_size_t, [_I] * 12),
    "forge_int8_conv2d_forward": (_I, [_P, _P, _P, _P, _P] + [_I] * 13 + [_P, _P]),
    "forge_int8_conv2d_nhwc_s32": (_I, [_P, _P, _P] + [_I] * 13 + [_P]),
    "forge_int8_conv2d_nhwc_dequant": (_I, [_P, _P, _P, _P, _P, _P] + [_I] * 13 + [_P]),
    "forge_quantize_weight_rows": (_I, [_P, _I, _P, _P, _I, _I, _P]),
    "forge_prepare_sparse_weight": (_I, [_P, _I, _P, _P, _P, _I, _I, _P]),
    "forge_int8_conv_transpose2d_k2s2_workspace_size": (ctypes.c_size_t, [_I] * 4),
    "forge_int8_conv_transpose2d_k2s2_forward": (_I, [_P] * 5 + [_I] * 5 + [_P, _P]),
    "forge_int8_depthwise_conv2d_forward": (_I, [_P] * 5 + [_I] * 12 + [_P]),
    "forge_quantize_weight_int4": (_I, [_P, _I, _P, _P, _I, _I, _I, _P]),
    "forge_pack_weight_int4": (_I, [_P, _P, _I, _I, _P]),
    "forge_int4_linear": (_I, [_P] * 5 + [_I] * 5 + [_P]),
    "forge_qk_norm_rope": (_I, [_P] * 13 + [_L] + [_I] * 6 + [_L] * 6 + [_F, _I, _I, _P]),
    "forge_prompt_attention": (_I, [_P] * 5 + [_I] * 5 + [_L] * 6 + [_F, _I, _I, _P]),
    "forge_cache_attention_workspace_size": (ctypes.c_size_t, [_I] * 5 + [_L]),
    "forge_cache_attention": (_I, [_P] * 7 + [_I] * 8 + [_F, _I, _P, ctypes.c_size_t, _P]),
    "forge_cache4_write": (_I, [_P] * 4 + [_I] * 5 + [_L] * 4 + [_I, _P]),
    "forge_cache4_read": (_I, [_P] * 4 + [_I] * 6 + [_P]),
    "forge_cache4_attention_workspace_size": (ctypes.c_size_t, [_I] * 5 + [_L]),
    "forge_cache4_attention": (_I, [_P] * 6 + [_I] * 8 + [_F, _I, _P, ctypes.c_size_t, _P]),
    "forge_beam_select_workspace_size": (ctypes.c_size_t, [_I] * 4),
    "forge_beam_select": (_I, [_P] * 3 + [_I] + [_P] * 3 + [_I] * 4 + [_L] * 2 + [_I, _P, ctypes.c_size_t, _P]),
    "forge_fork_pages_workspace_size": (ctypes.c_size_t, [_I] * 2),
    "forge_fork_pages": (_I, [_P] * 10 + [_I] * 5 + [_P, ctypes.c_size_t, _P]),
    "forge_copy_pages": (_I, [_P, _I, _L, _I, _P, _P, _I, _P]),
}

_lib = None


class ForgeError(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    """Returns the loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ForgeError(
                f"forge_amd native library not found at {LIB_PATH}; "
                "build it with `python -m forge_amd.build` (hipcc, gfx950)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


_calls = None


def calls():
    """The compiled calls of the decoder-attention operators (csrc/torch_calls.cpp), linked to the library."""
    global _calls
    if _calls is None:
        import importlib.machinery
        import importlib.util

        import torch  # noqa: F401  (its libraries, which the module needs)
        load()
        if not os.path.exists(BINDING_PATH):
            raise ForgeError(f"forge_amd binding not found at {BINDING_PATH}; build it with `python -m forge_amd.build`")
        loader = importlib.machinery.ExtensionFileLoader("forge_torch", BINDING_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("forge_torch", loader))
        loader.exec_module(module)
        _calls = module
    return _calls


def check(status: int, what: str = "") -> None:
    if status != FORGE_OK:
        msg = load().forge_status_string(status)
        raise ForgeError(f"{what}: status {status} ({msg.decode() if msg else '?'})")
