"""Host-side mirror of edge_maskgit's backend interface over libmgcuda.so.

``CudaRuntime`` mirrors ``mg::OpenCLRuntime`` (include/mg-opencl.hpp:23-58) for the MaskGIT
transformer graph: construct once per device, call ``forward`` (the ``TransformerFwd``
callback of include/mg-generate.hpp:15) once per decode step, optionally profile per op type.
The kernel-level functions (``quantize_act``, ``QWeight.qgemm``, ``layernorm_affine``,
``flash_attn``, ``embed``, ``gemm_f32``) take CUDA torch tensors and call the C ABI directly;
torch is only used for device memory and streams.
"""
from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass

import numpy as np

from ._lib import AttentionArgs, MgcError, check, lib
from ._lib import LogitControls as _LogitControls

__all__ = ["CudaRuntime", "VqganDecoder", "QWeight", "MgcError", "pack_q8_0", "pack_q4_k", "dequant", "tp_unique_id",
           "quantize_act", "gemm_f32", "layernorm_affine", "flash_attn", "embed", "device_error",
           "linear", "attention", "logits_adjust", "LogitControls", "F32", "F16", "BF16", "Q8_0", "Q4_K"]

F32, F16, Q8_0, Q4_K, BF16 = 0, 1, 8, 12, 30


def _ptr(a) -> C.c_void_p:
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        return C.c_void_p(a.ctypes.data)
    return C.c_void_p(a.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _cuda_f32(t, name):
    import torch
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
        raise MgcError(f"{name} must be a contiguous float32 CUDA tensor")
    return t


# ----------------------------------------------------------------- block formats (host)
def pack_q8_0(w: np.ndarray) -> np.ndarray:
    """[N][K] f32 -> GGUF Q8_0 bytes (tools/convert_to_gguf.py:109-124)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    N, K = w.shape
    out = np.empty(N * K // 32 * 34, np.uint8)
    check(lib.mgc_pack_q8_0(_ptr(w), N, K, _ptr(out)), "pack_q8_0")
    return out


def pack_q4_k(w: np.ndarray) -> np.ndarray:
    """[N][K] f32 -> GGUF Q4_K bytes (tools/convert_to_gguf.py:68-106)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    N, K = w.shape
    out = np.empty(N * K // 256 * 144, np.uint8)
    check(lib.mgc_pack_q4_k(_ptr(w), N, K, _ptr(out)), "pack_q4_k")
    return out


def dequant(wtype: int, blocks: np.ndarray, N: int, K: int) -> np.ndarray:
    """GGUF blocks -> [N][K] f32 (DEQ_Q8 / deq_q4k_elem of mg-opencl.cpp)."""
    blocks = np.ascontiguousarray(blocks, dtype=np.uint8)
    out = np.empty((N, K), np.float32)
    check(lib.mgc_dequant(wtype, _ptr(blocks), N, K, _ptr(out)), "dequant")
    return out


def device_error() -> int:
    """Read and clear the device error word set by kernels whose bounded waits expired."""
    return int(lib.mgc_device_error())


# ----------------------------------------------------------------- kernel-level ops
def quantize_act(x, want_sum: bool = False):
    """k_quantize_q8: x [M][K] -> (qx int8 [M][K], dx f32 [M][K/32], sumx int32 | None)."""
    import torch
    _cuda_f32(x, "x")
    M, K = x.shape
    qx = torch.empty((M, K), dtype=torch.int8, device=x.device)
    dx = torch.empty((M, K // 32), dtype=torch.float32, device=x.device)
    sx = torch.empty((M, K // 32), dtype=torch.int32, device=x.device) if want_sum else None
    check(lib.mgc_quantize_act(_ptr(x), M, K, _ptr(qx), _ptr(dx), _ptr(sx), _stream()), "quantize_act")
    return qx, dx, sx


class QWeight:
    """A Q8_0 / Q4_K (or F32) [N][K] weight resident on the current CUDA device."""

    def __init__(self, wtype: int, data: np.ndarray, N: int, K: int):
        data = np.ascontiguousarray(data)
        h = C.c_void_p()
        check(lib.mgc_qweight_create(wtype, _ptr(data), N, K, C.byref(h)), "qweight_create")
        self._h, self.wtype, self.N, self.K = h, wtype, N, K

    def qgemm(self, x, bias=None, act: int = 0, resid=None, out=None):
        """y = act(W.x + bias) + resid, the MulMat(q) dispatch of mg-opencl.cpp:1381-1399."""
        import torch
        _cuda_f32(x, "x")
        M = x.shape[0]
        if x.shape[1] != self.K:
            raise MgcError(f"x has {x.shape[1]} columns, weight K = {self.K}")
        y = out if out is not None else torch.empty((M, self.N), dtype=torch.float32, device=x.device)
        check(lib.mgc_qgemm(self._h, _ptr(x), M, _ptr(bias), act, _ptr(resid), _ptr(y), _stream()), "qgemm")
        return y

    def close(self):
        if self._h:
            lib.mgc_qweight_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def gemm_f32(w, x, bias=None, act: int = 0, resid=None):
    import torch
    N, K = w.shape
    M = x.shape[0]
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(lib.mgc_gemm_f32(_ptr(w), _ptr(x), M, N, K, _ptr(bias), act, _ptr(resid), _ptr(y), _stream()),
          "gemm_f32")
    return y


def layernorm_affine(x, gamma, beta, eps: float = 1e-12):
    import torch
    rows, D = x.shape
    y = torch.empty_like(x)
    check(lib.mgc_layernorm_affine(_ptr(x), _ptr(gamma), _ptr(beta), rows, D, eps, _ptr(y), _stream()),
          "layernorm_affine")
    return y


def flash_attn(qkv, B: int, S: int, H: int, Dh: int, scale: float):
    import torch
    y = torch.empty((B * S, H * Dh), dtype=torch.float32, device=qkv.device)
    check(lib.mgc_flash_attn(_ptr(qkv), B, S, H, Dh, scale, _ptr(y), _stream()), "flash_attn")
    return y


def embed(tok, pos, tokens, B: int, S: int):
    import torch
    V, E = tok.shape
    y = torch.empty((B * S, E), dtype=torch.float32, device=tok.device)
    check(lib.mgc_embed(_ptr(tok), V, _ptr(pos), E, _ptr(tokens), B, S, _ptr(y), _stream()), "embed")
    return y


# ----------------------------------------------------------------- 16-bit operators
# The checks below look at each tensor's type, device and gradient flag in one condition and
# explain only what failed: a small call is as long as its host side.
_CODE: dict = {}     # torch dtype -> code, filled with torch's names on the first call
_torch = None
# mgc_attention_args; mgc_attention takes its address
_ATTN_PACK = struct.Struct("8i4Q12q2f2Q2i5Q2Q")
assert _ATTN_PACK.size == C.sizeof(AttentionArgs)


def _load_torch():
    global _torch, _device, _raw_stream, _forward_ad, _is_tracing
    import torch
    import torch.autograd.forward_ad as _forward_ad
    _CODE.update({torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32})
    _device, _raw_stream, _is_tracing = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch._C._is_tracing
    _torch = torch
    return torch


def _only_values(**tensors):
    """Refuses what would be lost: these operators read their arguments' memory, so a forward-mode
    tangent does not pass through them, and a trace would hold an output that nothing fills."""
    if _is_tracing():
        raise MgcError("this operator cannot be recorded by torch.jit.trace")
    for name, t in tensors.items():
        if isinstance(t, _torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise MgcError(f"{name} carries a forward-mode tangent, which this operator does not pass on")


def _code_of(t, name, f32: bool = False) -> int:
    if _torch is None:
        _load_torch()
    code = _CODE.get(getattr(t, "dtype", None))
    if code is None or (code == F32 and not f32):
        raise MgcError(f"{name} must be {'float32, ' if f32 else ''}float16 or bfloat16, not {getattr(t, 'dtype', type(t))}")
    return code


def _refuse(t, name, dtype, index):
    torch = _torch or _load_torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
        raise MgcError(f"{name} must be a CUDA tensor" + (f" on device {index}" if index >= 0 else ""))
    if t.dtype != dtype:
        raise MgcError(f"{name} must be {dtype}, not {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise MgcError(f"{name} requires a gradient, which this operator does not give (use torch.no_grad())")


def _operand(t, name, dtype, index):
    """Checks a tensor that goes to the library by its address."""
    if t.__class__.__name__ != "Tensor" or t.dtype is not dtype or index < 0 or t.get_device() != index or t.requires_grad:
        _refuse(t, name, dtype, index)
    return t


def _vector(t, name, dtype, index, shape):
    """Address of an optional contiguous tensor of exactly this shape (0 for None)."""
    if t is None:
        return None
    _operand(t, name, dtype, index)
    if t.shape != shape or not t.is_contiguous():
        raise MgcError(f"{name} must be contiguous with shape {list(shape)}, not {list(t.shape)}")
    return t.data_ptr()


def _matrix(t, name, dtype, index):
    """Row stride of a 2-D tensor whose last axis is contiguous."""
    _operand(t, name, dtype, index)
    if t.dim() != 2:
        raise MgcError(f"{name} must have two axes, not {t.dim()}")
    ld, one = t.stride()
    if one != 1 and t.shape[1] > 1:
        raise MgcError(f"{name}'s last axis must be contiguous")
    return ld


def _elsewhere(index, what, fn, *args):
    """Calls the library with device `index` made current, on torch's stream there."""
    with _torch.cuda.device(index):
        check(fn(*args, _raw_stream(index)), what)


def linear(x, w, bias=None, act: int = 0, resid=None, out=None):
    """y = act(x W^T + bias) + resid in f16 / bf16 (mgc_linear): x [M][K], w [N][K], resid and y
    [M][N], bias f32 [N]; act 0 none, 1 erf-GELU, 2 SiLU; summed in f32, rounded once.  Rows may be
    strided; K and the row strides of x and w are multiples of 8.  `out` may be `resid`."""
    code = _CODE.get(getattr(x, "dtype", None)) or _code_of(x, "x")
    if _forward_ad._current_level >= 0 or _is_tracing():
        _only_values(x=x, w=w, bias=bias, resid=resid, out=out)
    dt, index = x.dtype, x.get_device()
    if index < 0 or w.dtype is not dt or w.get_device() != index or x.requires_grad or w.requires_grad or \
            not (x.dim() == w.dim() == 2):
        _matrix(x, "x", dt, index)
        _matrix(w, "w", dt, index)
    (M, K), (N, Kw) = x.shape, w.shape
    (ldx, one_x), (ldw, one_w) = x.stride(), w.stride()
    if (one_x != 1 or one_w != 1) and K > 1:
        raise MgcError("the last axes of x and w must be contiguous")
    if Kw != K:
        raise MgcError(f"x has {K} columns, w has {Kw}")
    if (M | N | K) >> 31:   # (ctypes would keep the low 32 bits)
        raise MgcError(f"linear: sizes must be below 2^31, not {[M, N, K]}")
    bias_p = _vector(bias, "bias", _torch.float32, index, (N,)) if bias is not None else None
    resid_p, ldr = None, 0
    if resid is not None:
        ldr = _matrix(resid, "resid", dt, index)
        resid_p = resid.data_ptr()
        if resid.shape != (M, N):
            raise MgcError(f"resid must have shape {[M, N]}, not {list(resid.shape)}")
    if out is None:
        out, ldy = x.new_empty((M, N)), N
    else:
        ldy = _matrix(out, "out", dt, index)
        if out.shape != (M, N):
            raise MgcError(f"out must have shape {[M, N]}, not {list(out.shape)}")
    if _device() != index:
        _elsewhere(index, "linear", lib.mgc_linear, code, x.data_ptr(), ldx, w.data_ptr(), ldw, M, N, K, bias_p, act,
                   resid_p, ldr, out.data_ptr(), ldy)
    elif lib.mgc_linear(code, x.data_ptr(), ldx, w.data_ptr(), ldw, M, N, K, bias_p, act, resid_p, ldr, out.data_ptr(), ldy,
                        _raw_stream(index)):
        check(-1, "linear")
    return out


def _heads(t, name, dtype, index):
    """Strides of a [batch][position][head][D] tensor."""
    _operand(t, name, dtype, index)
    if t.dim() != 4:
        raise MgcError(f"{name} must have four axes, not {t.dim()}")
    st = t.stride()
    if st[3] != 1 and t.shape[3] > 1:
        raise MgcError(f"{name}'s last axis must be contiguous")
    return st


def attention(q, k, v, scale: float | None = None, cap: float = 0.0, slopes=None, dist_bias=None, causal: bool = False,
              prefix=None, k_len=None, q_pos=None, doc_q=None, doc_k=None, out=None):
    """Attention with shaped scores in f16 / bf16 (mgc_attention).

    q [B][Sq][Hq][D], k and v [B][Sk][Hkv][D] (D a multiple of 8 up to 128, the last axis
    contiguous, the other strides multiples of 8) -> out like q.  With p = q_pos[b] + i (default
    Sk - Sq + i):
        s = scale * q.k;  cap > 0: s = cap tanh(s / cap);  s -= slopes[h] |p - j|
        s += dist_bias[h][clamp(j - p, -R, R) + R]     (dist_bias f32 [Hq][2 R + 1])
    over the keys j < k_len[b] that are j <= p or j < prefix[b] if causal, with doc_q[b][i] ==
    doc_k[b][j] >= 0 if given.  A query that sees no key gives zeros.  scale defaults to D ** -0.5;
    cap is 0 or from 2^-10 to 2^10; slopes f32 [Hq]; prefix, k_len, q_pos int32 [B]; doc_q, doc_k int32 [B][Sq], [B][Sk]."""
    code = _CODE.get(getattr(q, "dtype", None)) or _code_of(q, "q")
    if _forward_ad._current_level >= 0 or _is_tracing():
        _only_values(q=q, k=k, v=v, slopes=slopes, dist_bias=dist_bias, out=out)
    dt, index = q.dtype, q.get_device()
    if index < 0 or not (k.dtype is dt and v.dtype is dt and k.get_device() == index and v.get_device() == index) or \
            q.requires_grad or k.requires_grad or v.requires_grad or not (q.dim() == k.dim() == v.dim() == 4):
        for t, name in ((q, "q"), (k, "k"), (v, "v")):
            _heads(t, name, dt, index)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    B, Sq, Hq, D = q.shape
    Bk, Sk, Hkv, Dk = k.shape
    if (qs[3] != 1 or ks[3] != 1 or vs[3] != 1) and D > 1:
        raise MgcError("the last axes of q, k and v must be contiguous")
    if k.shape != v.shape or Bk != B or Dk != D:
        raise MgcError(f"k and v must be [{B}][Sk][Hkv][{D}], not {list(k.shape)} and {list(v.shape)}")
    i32, reach = _torch.int32, 0
    slopes_p = table_p = prefix_p = k_len_p = q_pos_p = doc_q_p = doc_k_p = None
    if slopes is not None:
        slopes_p = _vector(slopes, "slopes", _torch.float32, index, (Hq,))
    if dist_bias is not None:
        reach = dist_bias.shape[-1] // 2
        table_p = _vector(dist_bias, "dist_bias", _torch.float32, index, (Hq, 2 * reach + 1))
    if prefix is not None:
        if not causal:
            raise MgcError("prefix is for causal attention")
        prefix_p = _vector(prefix, "prefix", i32, index, (B,))
    if k_len is not None:
        k_len_p = _vector(k_len, "k_len", i32, index, (B,))
    if q_pos is not None:
        q_pos_p = _vector(q_pos, "q_pos", i32, index, (B,))
    if doc_q is not None:
        doc_q_p = _vector(doc_q, "doc_q", i32, index, (B, Sq))
    if doc_k is not None:
        doc_k_p = _vector(doc_k, "doc_k", i32, index, (B, Sk))
    if out is None:
        out, os = q.new_empty((B, Sq, Hq, D)), (Sq * Hq * D, Hq * D, D)
    else:
        os = _heads(out, "out", dt, index)
        if out.shape != q.shape:
            raise MgcError(f"out must have shape {list(q.shape)}, not {list(out.shape)}")
    head = (code, B, Sq, Sk, Hq, Hkv, D, 1 if causal else 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os[0], os[1], os[2],
            D ** -0.5 if scale is None else scale, cap, slopes_p or 0, table_p or 0, reach, 0, prefix_p or 0, k_len_p or 0,
            q_pos_p or 0, doc_q_p or 0, doc_k_p or 0)
    if _device() != index:   # (the split follows the current device's size)
        with _torch.cuda.device(index):
            _attention(index, q, head)
    else:
        _attention(index, q, head)
    return out


def _attention(index, q, head):
    try:
        args = _ATTN_PACK.pack(*head, 0, 0)
    except (struct.error, OverflowError) as e:   # beyond what the call's struct holds
        raise MgcError(f"attention: a size, scale or cap is out of range ({e})") from None
    need = C.c_uint64()
    rc = lib.mgc_attention_workspace(args, C.byref(need))
    if rc == 0:
        if need.value:   # from torch's allocator: this stream's (or this capture's) own memory
            ws = _torch.empty(need.value, dtype=_torch.uint8, device=q.device)
            args = _ATTN_PACK.pack(*head, ws.data_ptr(), need.value)
        rc = lib.mgc_attention(args, _raw_stream(index))
    if rc != 0:
        check(rc, "attention")


def logits_adjust(logits, history=None, hist_len=None, penalties=None, bias=None, allowed=None, out=None):
    """Penalties for repeated tokens, a bias and a bit mask on logits [R][V] (mgc_logits_adjust).

    For a token that row r's history (its first hist_len[r] values) holds c > 0 times,
    z = z > 0 ? z / rep : z * rep and z -= freq * c + pres; then z += bias[v], and -inf where bit
    v % 32 of allowed[v // 32] is 0.  logits f32, f16 or bf16; history int32 [R][L], hist_len int32
    [R], penalties f32 [R][3] = (rep, freq, pres), bias f32 [R][V], allowed int32 [R][(V + 31) // 32].
    One-axis history, penalties, bias or allowed are shared by all rows.  `out` may be `logits`."""
    code = _code_of(logits, "logits", f32=True)
    if _forward_ad._current_level >= 0 or _is_tracing():
        _only_values(logits=logits, penalties=penalties, bias=bias, out=out)
    dt, index = logits.dtype, logits.get_device()
    ld = _matrix(logits, "logits", dt, index)
    R, V = logits.shape
    i32, f32 = _torch.int32, _torch.float32

    def table(t, name, dtype, width):   # (pointer, row stride), 0 = one row for all
        if t.dim() == 1:
            _operand(t, name, dtype, index)
            if t.shape[0] > 1 and t.stride(0) != 1:
                raise MgcError(f"{name} must be contiguous")
            cols, stride = t.shape[0], 0
        else:
            stride = _matrix(t, name, dtype, index)
            rows, cols = t.shape
            if rows != R:
                raise MgcError(f"{name} must have {R} rows, not {rows}")
            if R == 1:
                stride = 0
        if cols != width:
            raise MgcError(f"{name} must have {width} columns, not {cols}")
        return t.data_ptr(), stride

    hist_p = len_p = pen_p = bias_p = allowed_p = None
    L = ld_h = ld_p = ld_b = ld_a = 0
    if (history is None) != (penalties is None):
        raise MgcError("history and penalties are given together")
    if history is not None:
        L = history.shape[-1]
        hist_p, ld_h = table(history, "history", i32, L)
        pen_p, ld_p = table(penalties, "penalties", f32, 3)
        if hist_len is not None:
            len_p = _vector(hist_len, "hist_len", i32, index, (R,))
        if L == 0:   # an empty history: nothing is repeated
            hist_p = pen_p = None
    elif hist_len is not None:
        raise MgcError("hist_len is for a history")
    if bias is not None:
        bias_p, ld_b = table(bias, "bias", f32, V)
    if allowed is not None:
        allowed_p, ld_a = table(allowed, "allowed", i32, (V + 31) // 32)
    if (R | V | L) >> 31:   # (ctypes would keep the low 32 bits)
        raise MgcError(f"logits_adjust: sizes must be below 2^31, not {[R, V, L]}")
    if out is None:
        out, ld_o = logits.new_empty((R, V)), V
    else:
        ld_o = _matrix(out, "out", dt, index)
        if out.shape != logits.shape:
            raise MgcError(f"out must have shape {list(logits.shape)}, not {list(out.shape)}")
    if _device() != index:
        _elsewhere(index, "logits_adjust", lib.mgc_logits_adjust, code, logits.data_ptr(), ld, R, V, hist_p, ld_h, L, len_p,
                   pen_p, ld_p, bias_p, ld_b, allowed_p, ld_a, out.data_ptr(), ld_o)
    elif lib.mgc_logits_adjust(code, logits.data_ptr(), ld, R, V, hist_p, ld_h, L, len_p, pen_p, ld_p, bias_p, ld_b,
                               allowed_p, ld_a, out.data_ptr(), ld_o, _raw_stream(index)):
        check(-1, "logits_adjust")
    return out


# ----------------------------------------------------------------- runtime
@dataclass
class HParams:
    n_layer: int
    n_head: int
    n_embd: int
    n_ffn: int
    head_dim: int
    vocab_size: int
    n_tokens: int
    mask_token_id: int
    codebook_size: int
    wtype: int


@dataclass
class OpProfile:   # include/mg-opencl.hpp:17-21
    op: str
    count: int
    ms: float


@dataclass
class LogitControls:
    """What generate() does to the logits of the codes before each draw (mgc_logit_controls):
    penalties against the codes an image already holds, a bias [codebook], and allowed codes as
    truth values [codebook] or, one row per grid cell, [n_tokens][codebook].  The bias is finite,
    repetition from 2^-60 to 2^60, frequency and presence at most 2^60."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: np.ndarray | None = None
    allowed: np.ndarray | None = None

    def _struct(self, codebook: int):
        """The C struct and the arrays that must outlive it."""
        bias = None
        if self.bias is not None:
            bias = np.ascontiguousarray(self.bias, np.float32)
            if bias.shape != (codebook,):
                raise MgcError(f"bias must have shape [{codebook}], not {list(bias.shape)}")
        bits, rows = None, 0
        if self.allowed is not None:
            a = np.atleast_2d(np.asarray(self.allowed, bool))
            if a.ndim != 2 or a.shape[1] != codebook:
                raise MgcError(f"allowed must have {codebook} columns, not shape {list(a.shape)}")
            rows = a.shape[0]
            a = np.pad(a, ((0, 0), (0, -codebook % 32)))
            bits = np.ascontiguousarray(np.packbits(a, axis=1, bitorder="little")).view("<u4")
        return _LogitControls(self.repetition, self.frequency, self.presence, _ptr(bias), _ptr(bits), rows), (bias, bits)


def tp_unique_id() -> bytes:
    """128-byte NCCL id for a tensor-parallel runtime group (make it on one rank, share it)."""
    buf = (C.c_uint8 * 128)()
    check(lib.mgc_tp_unique_id(buf), "tp_unique_id")
    return bytes(buf)


class CudaRuntime:
    """mg::OpenCLRuntime's counterpart for the MaskGIT transformer on one B200.

    tp=(rank, world, id) makes this process rank `rank` of a column-split tensor-parallel group
    of `world` GPUs (id from tp_unique_id() on one rank); all ranks then run every forward with
    the same inputs and each gets the full logits."""

    def __init__(self, gguf_path: str, max_rows: int = 257, device: int = 0, tp=None):
        h = C.c_void_p()
        if tp is None:
            check(lib.mgc_runtime_create(str(gguf_path).encode(), max_rows, device, C.byref(h)), "runtime_create")
        else:
            rank, world, uid = tp
            idb = (C.c_uint8 * 128).from_buffer_copy(uid)
            check(lib.mgc_runtime_create_tp(str(gguf_path).encode(), max_rows, device, rank, world, idb, C.byref(h)),
                  "runtime_create_tp")
        self._h = h
        hp = np.zeros(10, np.int32)
        check(lib.mgc_runtime_hparams(h, _ptr(hp)))
        self.hparams = HParams(*[int(v) for v in hp])
        self.max_rows = max_rows

    # --- OpenCLRuntime API
    def device_name(self) -> str:
        return lib.mgc_runtime_device_name(self._h).decode()

    def invalidate(self, _tensor=None) -> None:
        """Token inputs are uploaded on every forward, so nothing is cached to drop."""

    def profile_enable(self, on: bool) -> None:
        check(lib.mgc_profile_enable(self._h, int(on)))

    def profile_reset(self) -> None:
        check(lib.mgc_profile_reset(self._h))

    def kernel_count(self) -> int:
        """Kernels enqueued by the last forward."""
        return int(lib.mgc_runtime_kernel_count(self._h))

    def time_op(self, op: str, B: int, S: int, iters: int = 50) -> tuple[float, int]:
        """(ms per replay, kernels per replay) of a CUDA graph holding only the forward's
        launches of op class `op` (a profile_report name), replayed back to back."""
        ms, n = C.c_float(), C.c_int()
        check(lib.mgc_runtime_time_op(self._h, op.encode(), B, S, iters, C.byref(ms), C.byref(n)), "time_op")
        return float(ms.value), int(n.value)

    def profile_report(self) -> list[OpProfile]:
        buf = C.create_string_buffer(1 << 14)
        check(lib.mgc_profile_report(self._h, buf, len(buf)))
        rows = []
        for line in buf.value.decode().splitlines():
            name, n, ms = line.rsplit(" ", 2)
            rows.append(OpProfile(name, int(n), float(ms)))
        return rows

    # --- TransformerFwd
    def forward(self, tokens: np.ndarray, B: int | None = None, out: np.ndarray | None = None) -> np.ndarray:
        """tokens [B][S] int32 (host) -> logits [B*S][vocab] f32 (host).  `out` (optional) is a
        caller-owned C-contiguous float32 [B*S][vocab] buffer reused across calls, as the
        reference decode loop reuses its logits vector (mg-generate.cpp:55)."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        if tokens.ndim == 1:
            tokens = tokens[None]
        B, S = tokens.shape
        shape = (B * S, self.hparams.vocab_size)
        if out is None:
            out = np.empty(shape, np.float32)
        elif out.shape != shape or out.dtype != np.float32 or not out.flags.c_contiguous:
            raise ValueError(f"out must be a C-contiguous float32 array of shape {shape}")
        check(lib.mgc_transformer_forward(self._h, _ptr(tokens), B, S, _ptr(out)), "forward")
        return out

    def forward_dev(self, tokens_dev, logits_dev, B: int, S: int) -> None:
        """Device-resident forward on the runtime's stream (graph replay); not synchronised."""
        check(lib.mgc_transformer_forward_dev(self._h, _ptr(tokens_dev), B, S, _ptr(logits_dev)), "forward_dev")

    def forward_dump(self, tokens: np.ndarray):
        """Forward that also returns the 51 named verification tensors (MG_DUMP_NAMED)."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        if tokens.ndim == 1:
            tokens = tokens[None]
        B, S = tokens.shape
        hp = self.hparams
        R = B * S
        logits = np.empty((R, hp.vocab_size), np.float32)
        dump = np.empty(R * (hp.n_embd * (2 * hp.n_layer + 2) + hp.vocab_size), np.float32)
        check(lib.mgc_transformer_forward_dump(self._h, _ptr(tokens), B, S, _ptr(logits), _ptr(dump)),
              "forward_dump")
        return logits, split_named(dump, R, hp.n_layer, hp.n_embd, hp.vocab_size)

    def sync(self) -> None:
        check(lib.mgc_runtime_sync(self._h), "sync")

    @property
    def stream_handle(self) -> int:
        return int(lib.mgc_runtime_stream(self._h) or 0)

    def generate(self, class_ids, seeds, steps: int = 8, temperature: float = 4.5,
                 controls: LogitControls | None = None) -> np.ndarray:
        """generate() (src/mg-generate.cpp:53-123) for len(class_ids) images -> tokens [B][S].
        `controls` adjusts the logits before every draw."""
        cls = np.ascontiguousarray(class_ids, dtype=np.int32)
        sd = np.ascontiguousarray(seeds, dtype=np.uint64)
        B = cls.shape[0]
        if sd.size < B:
            raise MgcError(f"generate: {B} images need a seed each, not {sd.size}")
        out = np.empty((B, self.hparams.n_tokens + 1), np.int32)
        if controls is None:
            check(lib.mgc_generate(self._h, B, _ptr(cls), _ptr(sd), steps, temperature, _ptr(out)), "generate")
        else:
            c, _alive = controls._struct(self.hparams.codebook_size)
            check(lib.mgc_generate_with(self._h, B, _ptr(cls), _ptr(sd), steps, temperature, C.byref(c), _ptr(out)), "generate")
        return out

    def generate_images(self, vq: "VqganDecoder", class_ids, seeds, steps: int = 8,
                        temperature: float = 4.5) -> tuple[np.ndarray, np.ndarray]:
        """mg::generate end to end (mgc_generate_images): uint8 images [B][R][R][3] and the
        final token sequences [B][n_tokens + 1]."""
        cls = np.ascontiguousarray(class_ids, np.int32)
        sd = np.ascontiguousarray(seeds, np.uint64)
        B, R = len(cls), vq.resolution
        if sd.size < B:
            raise MgcError(f"generate_images: {B} images need a seed each, not {sd.size}")
        rgb = np.empty((B, R, R, 3), np.uint8)
        tok = np.empty((B, self.hparams.n_tokens + 1), np.int32)
        check(lib.mgc_generate_images(self._h, vq._h, B, _ptr(cls), _ptr(sd), steps, temperature, _ptr(rgb),
                                      _ptr(tok)), "generate_images")
        return rgb, tok

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib.mgc_runtime_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class VqganDecoder:
    """The VQGAN decoder (build_vqgan_decoder, include/mg-vqgan.hpp:12) on one B200.

    ``decode(grid)`` is the reference's VqganFwd callback (include/mg-generate.hpp:17): a token
    grid [n_tokens] (or a batch [n][n_tokens]) -> HWC float image [R][R][3] (or [n][R][R][3])."""

    def __init__(self, gguf_path: str, max_images: int = 1, device: int = 0):
        h = C.c_void_p()
        check(lib.mgc_vqgan_create(str(gguf_path).encode(), max_images, device, C.byref(h)), "vqgan_create")
        self._h = h
        info = [C.c_int(), C.c_int(), C.c_int()]
        check(lib.mgc_vqgan_info(h, *[C.byref(v) for v in info]))
        self.n_tokens, self.resolution, self.codebook_size = (v.value for v in info)
        self.max_images = max_images

    def decode(self, grid, out: np.ndarray | None = None) -> np.ndarray:
        g = np.ascontiguousarray(grid, np.int32)
        single = g.ndim == 1
        g = g.reshape(-1, self.n_tokens)
        R = self.resolution
        if out is None:
            out = np.empty((g.shape[0], R, R, 3), np.float32)
        check(lib.mgc_vqgan_decode(self._h, _ptr(g), g.shape[0], _ptr(out)), "vqgan_decode")
        return out[0] if single else out

    def decode_rgb8(self, grid) -> np.ndarray:
        """The bytes of the reference's mg::Image (clamp, * 255 + 0.5, truncate): uint8 HWC."""
        g = np.ascontiguousarray(grid, np.int32)
        single = g.ndim == 1
        g = g.reshape(-1, self.n_tokens)
        R = self.resolution
        out = np.empty((g.shape[0], R, R, 3), np.uint8)
        check(lib.mgc_vqgan_decode_rgb8(self._h, _ptr(g), g.shape[0], _ptr(out)), "vqgan_decode_rgb8")
        return out[0] if single else out

    def decode_device(self, grid_dev, out_dev, n_images: int) -> None:
        """Device tensors (int32 [n][n_tokens], float32 [n][R][R][3]) on the current torch stream."""
        check(lib.mgc_vqgan_decode_device(self._h, _ptr(grid_dev), n_images, _ptr(out_dev), _stream()),
              "vqgan_decode_device")

    def launches(self) -> int:
        return lib.mgc_vqgan_launches(self._h)

    def time_op(self, op: str, n_images: int = 1, iters: int = 20) -> tuple[float, int]:
        """(ms per replay, launches) of a graph of one kernel class of the decode."""
        ms, n = C.c_float(), C.c_int()
        check(lib.mgc_vqgan_time_op(self._h, op.encode(), n_images, iters, C.byref(ms), C.byref(n)), "vqgan_time_op")
        return ms.value, n.value

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib.mgc_vqgan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def named_tensor_names(n_layer: int) -> list[str]:
    """The 51 verification names of mg-transformer.cpp:48,91,98,105,109 in dump order."""
    names = ["embd_post_norm"]
    for i in range(n_layer):
        names += [f"blk.{i}.attn_post", f"blk.{i}.ffn_post"]
    return names + ["output_norm", "output_logits"]


def split_named(dump: np.ndarray, R: int, n_layer: int, E: int, V: int) -> dict:
    out, off = {}, 0
    for name in named_tensor_names(n_layer):
        w = V if name == "output_logits" else E
        out[name] = dump[off:off + R * w].reshape(R, w)
        off += R * w
    return out
