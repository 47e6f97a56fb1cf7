"""ctypes binding of libmgcuda.so (the C ABI declared in include/mgc.h).

The library is built in-tree by ``edge_maskgit_b200.build``.  There is no fallback: if the
shared object is missing, importing this module raises.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libmgcuda.so"

if not LIB_PATH.exists():
    raise ImportError(f"{LIB_PATH} is missing: run `python -m edge_maskgit_b200.build` "
                      "(the CUDA backend has no CPU fallback)")

lib = C.CDLL(str(LIB_PATH))

P = C.c_void_p
I = C.c_int
I64 = C.c_int64
F = C.c_float


class AttentionArgs(C.Structure):
    """mgc_attention_args"""
    _fields_ = [("dtype", C.c_int32), ("B", C.c_int32), ("Sq", C.c_int32), ("Sk", C.c_int32), ("Hq", C.c_int32),
                ("Hkv", C.c_int32), ("D", C.c_int32), ("causal", C.c_int32),
                ("q", P), ("k", P), ("v", P), ("out", P),
                ("q_stride", I64 * 3), ("k_stride", I64 * 3), ("v_stride", I64 * 3), ("out_stride", I64 * 3),
                ("scale", F), ("cap", F), ("slopes", P), ("dist_bias", P), ("dist_range", C.c_int32),
                ("reserved", C.c_int32), ("prefix", P), ("k_len", P), ("q_pos", P), ("doc_q", P), ("doc_k", P),
                ("workspace", P), ("workspace_bytes", C.c_uint64)]


class LogitControls(C.Structure):
    """mgc_logit_controls"""
    _fields_ = [("repetition", F), ("frequency", F), ("presence", F), ("bias", P), ("allowed", P),
                ("allowed_rows", C.c_int32)]


_SIGS = {
    "mgc_last_error": (C.c_char_p, []),
    "mgc_device_error": (I, []),
    "mgc_selftest_wait_timeout": (I, [I, P]),
    "mgc_pack_q8_0": (I, [P, I64, I64, P]),
    "mgc_pack_q4_k": (I, [P, I64, I64, P]),
    "mgc_dequant": (I, [I, P, I64, I64, P]),
    "mgc_quantize_act": (I, [P, I, I, P, P, P, P]),
    "mgc_qweight_create": (I, [I, P, I, I, C.POINTER(P)]),
    "mgc_qweight_destroy": (None, [P]),
    "mgc_qgemm": (I, [P, P, I, P, I, P, P, P]),
    "mgc_qgemm_noalloc": (I, [P, P, I, P, I, P, P, P]),
    "mgc_gemm_f32": (I, [P, P, I, I, I, P, I, P, P, P]),
    "mgc_layernorm_affine": (I, [P, P, P, I, I, F, P, P]),
    "mgc_flash_attn": (I, [P, I, I, I, I, F, P, P]),
    "mgc_embed": (I, [P, I, P, I, P, I, I, P, P]),
    "mgc_linear": (I, [I, P, I64, P, I64, I, I, I, P, I, P, I64, P, I64, P]),
    "mgc_attention_workspace": (I, [P, P]),   # AttentionArgs (by reference, or packed bytes), uint64
    "mgc_attention": (I, [P, P]),
    "mgc_selftest_attention_gives_up": (I, [P, P]),
    "mgc_logits_adjust": (I, [I, P, I64, I, I, P, I64, I, P, P, I64, P, I64, P, I64, P, I64, P]),
    "mgc_generate_with": (I, [P, I, P, P, I, F, C.POINTER(LogitControls), P]),
    "mgc_runtime_create": (I, [C.c_char_p, I, I, C.POINTER(P)]),
    "mgc_runtime_destroy": (None, [P]),
    "mgc_tp_unique_id": (I, [P]),
    "mgc_runtime_create_tp": (I, [C.c_char_p, I, I, I, I, P, C.POINTER(P)]),
    "mgc_runtime_hparams": (I, [P, P]),
    "mgc_runtime_device_name": (C.c_char_p, [P]),
    "mgc_transformer_forward": (I, [P, P, I, I, P]),
    "mgc_transformer_forward_dev": (I, [P, P, I, I, P]),
    "mgc_transformer_forward_dump": (I, [P, P, I, I, P, P]),
    "mgc_runtime_sync": (I, [P]),
    "mgc_runtime_stream": (P, [P]),
    "mgc_generate": (I, [P, I, P, P, I, F, P]),
    "mgc_runtime_kernel_count": (I, [P]),
    "mgc_runtime_time_op": (I, [P, C.c_char_p, I, I, I, C.POINTER(F), C.POINTER(I)]),
    "mgc_profile_enable": (I, [P, I]),
    "mgc_profile_reset": (I, [P]),
    "mgc_profile_report": (I, [P, C.c_char_p, C.c_size_t]),
    "mgc_vqgan_create": (I, [C.c_char_p, I, I, C.POINTER(P)]),
    "mgc_vqgan_info": (I, [P, P, P, P]),
    "mgc_vqgan_decode": (I, [P, P, I, P]),
    "mgc_vqgan_decode_device": (I, [P, P, I, P, P]),
    "mgc_vqgan_decode_rgb8": (I, [P, P, I, P]),
    "mgc_generate_images": (I, [P, P, I, P, P, I, F, P, P]),
    "mgc_vqgan_launches": (I, [P]),
    "mgc_vqgan_time_op": (I, [P, C.c_char_p, I, I, C.POINTER(F), C.POINTER(I)]),
    "mgc_vqgan_destroy": (None, [P]),
}

for _name, (_res, _args) in _SIGS.items():
    _fn = getattr(lib, _name)
    _fn.restype = _res
    _fn.argtypes = _args

EXPORTED = tuple(_SIGS)


class MgcError(RuntimeError):
    pass


def check(rc: int, what: str = "") -> None:
    if rc != 0:
        msg = lib.mgc_last_error().decode(errors="replace")
        raise MgcError(f"{what}: {msg}" if what else msg)
