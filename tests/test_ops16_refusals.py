"""CPU: what mgc_linear, mgc_attention, mgc_logits_adjust and their Python forms refuse, before
anything reaches a GPU."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20   # an aligned address that is never read: every call here is refused first


def _err(lib):
    return lib.mgc_last_error().decode()


LINEAR = dict(dtype=1, x=A, ldx=64, w=A, ldw=64, M=4, N=8, K=64, bias=None, act=0, resid=None, ldr=0, y=A, ldy=8, st=None)


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=0), "dtype"), (dict(dtype=8), "dtype"), (dict(M=-1), "size"), (dict(K=60), "K"), (dict(K=0), "K"),
    (dict(act=3), "act"), (dict(act=-1), "act"), (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(x=A + 2), "aligned"),
    (dict(w=A + 8), "aligned"), (dict(y=A + 1), "aligned"), (dict(bias=A + 2), "aligned"), (dict(ldx=63), "ldx"),
    (dict(ldx=68), "ldx"), (dict(ldw=56), "ldx and ldw"), (dict(ldy=7), "ldy"), (dict(resid=A, ldr=7), "ldy and ldr"),
    (dict(resid=A, y=A, ldr=8, ldy=16), "in place"),
])
def test_linear_refuses(bad, word):
    from edge_maskgit_b200._lib import lib
    assert lib.mgc_linear(*dict(LINEAR, **bad).values()) == -1
    assert word in _err(lib)


def test_empty_calls_are_no_ops():
    from edge_maskgit_b200._lib import AttentionArgs, lib
    assert lib.mgc_linear(*dict(LINEAR, M=0, x=None, y=None).values()) == 0
    assert lib.mgc_linear(*dict(LINEAR, N=0).values()) == 0
    assert lib.mgc_logits_adjust(*dict(LOGITS, R=0, z=None).values()) == 0
    assert lib.mgc_logits_adjust(*dict(LOGITS, V=0).values()) == 0
    for change in (dict(B=0), dict(Sq=0)):
        args = _attn(**change)
        need = C.c_uint64(7)
        assert lib.mgc_attention_workspace(C.byref(args), C.byref(need)) == 0 and need.value == 0
        assert lib.mgc_attention(C.byref(args), None) == 0
    assert isinstance(args, AttentionArgs)


LOGITS = dict(dtype=0, z=A, ld=100, R=2, V=100, hist=A, ldh=5, L=5, hist_len=None, pen=A, ldp=3, bias=None, ldb=0,
              allowed=None, lda=0, out=A, ldo=100, st=None)


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=12), "dtype"), (dict(R=-1), "size"), (dict(V=-1), "size"), (dict(L=-1), "size"), (dict(z=None), "NULL"),
    (dict(out=None), "NULL"), (dict(pen=None), "together"), (dict(hist=None), "together"), (dict(z=A + 2), "aligned"),
    (dict(hist=A + 1), "aligned"), (dict(allowed=A + 2), "aligned"), (dict(ld=99, ldo=99), "ld"), (dict(out=2 * A, ldo=99), "ld_out"),
    (dict(ldo=104), "in place"), (dict(ldh=4), "ld_history"), (dict(ldp=2), "ld_penalties"), (dict(bias=A, ldb=99), "ld_bias"),
    (dict(allowed=A, lda=3), "ld_allowed"),
])
def test_logits_adjust_refuses(bad, word):
    from edge_maskgit_b200._lib import lib
    assert lib.mgc_logits_adjust(*dict(LOGITS, **bad).values()) == -1
    assert word in _err(lib)


def _attn(**kw):
    from edge_maskgit_b200._lib import AttentionArgs
    a = AttentionArgs(dtype=1, B=2, Sq=3, Sk=5, Hq=4, Hkv=2, D=64, causal=0, q=A, k=A, v=A, out=A, scale=0.125)
    a.q_stride[:] = a.out_stride[:] = [3 * 256, 256, 64]
    a.k_stride[:] = a.v_stride[:] = [5 * 128, 128, 64]
    for name, value in kw.items():
        if name.endswith("_stride"):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=0), "dtype"), (dict(B=-1), "size"), (dict(Sk=-1), "size"), (dict(Hkv=3), "Hq"), (dict(Hkv=0), "Hq"),
    (dict(D=0), "D must"), (dict(D=60), "D must"), (dict(D=136), "D must"), (dict(causal=2), "causal"),
    (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"),
    (dict(dist_range=-1), "dist_range"), (dict(doc_q=A), "together"), (dict(reserved=1), "reserved"),
    (dict(Sq=1 << 29), "too large"),
])
def test_attention_refuses_sizes(bad, word):
    from edge_maskgit_b200._lib import lib
    need = C.c_uint64()
    for rc in (lib.mgc_attention_workspace(C.byref(_attn(**bad)), C.byref(need)), lib.mgc_attention(C.byref(_attn(**bad)), None)):
        assert rc == -1 and word in _err(lib)


@pytest.mark.parametrize("bad,word", [
    (dict(cap=2.0 ** -11), "cap"), (dict(cap=2.0 ** 11), "cap"), (dict(scale=2.0 ** 101), "scale"),
    (dict(scale=-2.0 ** 101), "scale"), (dict(scale=2.0 ** 13, cap=2.0 ** -8), "scale must be at most 2^20 cap"),
])
def test_attention_refuses_constants_out_of_range(bad, word):
    """A cap far above 1024 would carry its rounding into the scores; a scale far above the cap overflows."""
    from edge_maskgit_b200._lib import lib
    need = C.c_uint64()
    assert lib.mgc_attention_workspace(C.byref(_attn(**bad)), C.byref(need)) == -1 and word in _err(lib)


def test_null_structs_are_refused():
    from edge_maskgit_b200._lib import lib
    assert lib.mgc_attention(None, None) == -1 and "NULL" in _err(lib)
    assert lib.mgc_attention_workspace(None, C.byref(C.c_uint64())) == -1


def test_python_forms_refuse():
    from edge_maskgit_b200 import runtime as rt
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(8, 64, dtype=torch.float16)
    with pytest.raises(rt.MgcError, match="CUDA"):
        rt.linear(x, w)
    with pytest.raises(rt.MgcError, match="float16 or bfloat16"):
        rt.linear(x.float(), w)
    with pytest.raises(rt.MgcError, match="CUDA"):
        rt.logits_adjust(torch.zeros(2, 5))
    with pytest.raises(rt.MgcError, match="float32, float16 or bfloat16"):
        rt.logits_adjust(torch.zeros(2, 5, dtype=torch.float64))
    q = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(rt.MgcError, match="CUDA"):
        rt.attention(q, q, q)


def test_logit_controls_struct():
    import numpy as np
    from edge_maskgit_b200 import runtime as rt
    allowed = np.zeros((3, 40), bool)
    allowed[0, 0] = allowed[1, 31] = allowed[2, 32] = True
    c, (bias, bits) = rt.LogitControls(repetition=1.5, bias=np.arange(40.0), allowed=allowed)._struct(40)
    assert bits.tolist() == [[1, 0], [1 << 31, 0], [0, 1]] and c.allowed_rows == 3 and bias.dtype == np.float32
    with pytest.raises(rt.MgcError, match="columns"):
        rt.LogitControls(allowed=np.ones(39, bool))._struct(40)
    with pytest.raises(rt.MgcError, match="bias"):
        rt.LogitControls(bias=np.ones(39))._struct(40)
