"""GPU: the 16-bit operators (mgc_linear, mgc_attention, mgc_logits_adjust) against plain forms in
64 bits.

Tolerances are derived, not fitted.  A result rounded to type t is off by half a step, eps / 2
relative.  Sums run in f32 on tensor cores, whose adders may drop bits below 2^-22 of the largest
term: n terms are off by at most n 2^-22 sum|terms|.  Attention also rounds each probability to t
before its product with v: another eps / 2 of sum p |v|."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U22 = 2.0 ** -22


@pytest.fixture(scope="module", autouse=True)
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield torch.device("cuda:0")
    from edge_maskgit_b200 import runtime as rt
    torch.cuda.synchronize()
    assert rt.device_error() == 0


def half_step(dt):
    return torch.finfo(dt).eps / 2


def randn(*shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def within(y, ref, tol):
    """Elementwise |y - ref| <= tol, with infinities and NaN in the same places."""
    y, bad = y.double(), ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    assert torch.equal(y[bad & ~torch.isnan(ref)], ref[bad & ~torch.isnan(ref)])
    diff = torch.where(bad, 0.0, (y - torch.where(bad, 0.0, ref)).abs())
    worst = (diff - tol).max().item() if ref.numel() else 0.0
    assert not worst > 0, f"off by {diff.max().item():.3e}, {worst:.3e} over the tolerance"


# ------------------------------------------------------------------------------------ linear
def linear_ref(x, w, bias, act, resid):
    acc = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        acc, mag = acc + bias.double(), mag + bias.double().abs()
    y = acc
    if act == 1:
        y = acc * 0.5 * (1 + torch.erf(acc * math.sqrt(0.5)))
    elif act == 2:
        y = acc * torch.sigmoid(acc)
    # both activations change by at most 1.13 times their argument's change; their own f32
    # evaluation is off by a few 2^-22 of the argument
    tol = 1.13 * (x.shape[1] + 2) * U22 * mag + 4 * U22 * acc.abs()
    if resid is not None:
        y = y + resid.double()
        tol = tol + U22 * resid.double().abs()
    return y, tol + half_step(x.dtype) * (y.abs() + tol) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps


def check_linear(x, w, bias=None, act=0, resid=None, out=None):
    from edge_maskgit_b200 import runtime as rt
    ref, tol = linear_ref(x, w, bias, act, resid)
    y = rt.linear(x, w, bias=bias, act=act, resid=resid, out=out)
    assert y.dtype == x.dtype
    within(y, ref, tol)
    return y


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 8, 1), (1, 64, 128), (1, 4096, 4096), (3, 72, 130), (16, 768, 2304), (17, 768, 257),
                                   (33, 200, 300), (65, 1000, 77), (129, 768, 2025), (257, 768, 768), (300, 64, 16),
                                   (1025, 520, 2025), (2049, 768, 2304), (5, 8192, 64)])
def test_linear_shapes(dt, M, K, N):
    check_linear(randn(M, K, dtype=dt, seed=1), randn(N, K, dtype=dt, seed=2, std=K ** -0.5))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("M,N", [(1, 2025), (40, 2025), (257, 2304), (4099, 1033)])
@pytest.mark.parametrize("use_bias,use_resid", [(True, False), (False, True), (True, True)])
def test_linear_epilogue(dt, act, M, N, use_bias, use_resid):
    K = 264
    check_linear(randn(M, K, dtype=dt, seed=3), randn(N, K, dtype=dt, seed=4, std=3 * K ** -0.5),
                 bias=randn(N, dtype=F32, seed=5) if use_bias else None, act=act,
                 resid=randn(M, N, dtype=dt, seed=6) if use_resid else None)


@pytest.mark.parametrize("act", [1, 2])
@pytest.mark.parametrize("M,N", [(3, 64), (700, 2304), (8200, 2304)])
def test_linear_activation_near_the_largest_float(act, M, N):
    """Sums between half of float32's largest value and the largest: the activation is the value itself
    (or -0), not infinity.  One term of K = 8 is not 0, so the sum is exact."""
    from edge_maskgit_b200 import runtime as rt
    x, w = torch.zeros(M, 8, device="cuda", dtype=BF16), torch.zeros(N, 8, device="cuda", dtype=BF16)
    x[:, 0] = 2.0 ** 64
    w[0::2, 0], w[1::2, 0] = 1.5 * 2.0 ** 63, -1.5 * 2.0 ** 63
    y = rt.linear(x, w, act=act)
    assert torch.all(y[:, 0::2] == 1.5 * 2.0 ** 127) and torch.all(y[:, 1::2] == 0)


@pytest.mark.parametrize("M,N", [(7, 300), (2000, 2056)])
def test_linear_strided_rows_and_in_place_residual(M, N):
    K = 136
    x = randn(M, K + 24, dtype=BF16, seed=7)[:, 8:8 + K]
    w = randn(N, K + 8, dtype=BF16, seed=8, std=K ** -0.5)[:, :K]
    wide = randn(M, N + 5, dtype=BF16, seed=9)
    kept = wide.clone()
    y = wide[:, 2:2 + N]
    check_linear(x, w, resid=y.clone(), out=torch.empty_like(wide)[:, 1:1 + N])
    ref, tol = linear_ref(x, w, None, 0, y.clone())
    from edge_maskgit_b200 import runtime as rt
    rt.linear(x, w, resid=y, out=y)
    within(y, ref, tol)
    assert torch.equal(wide[:, :2], kept[:, :2]) and torch.equal(wide[:, 2 + N:], kept[:, 2 + N:])


def test_linear_special_values():
    from edge_maskgit_b200 import runtime as rt
    x, w = randn(4, 64, dtype=F16, seed=10), randn(40, 64, dtype=F16, seed=11)
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    w[:, 5] = w[:, 5].abs() + 1
    y = rt.linear(x, w)
    assert y[1].isnan().all() and (y[2] == math.inf).all()
    within(y[[0, 3]], *linear_ref(x[[0, 3]], w, None, 0, None))
    big = torch.full((1, 64), 300.0, device="cuda", dtype=F16)
    assert (rt.linear(big, big) == math.inf).all()   # 64 * 300^2 > 65504: rounds to infinity


# ------------------------------------------------------------------------------------ logits
def logits_ref(z, history=None, hist_len=None, penalties=None, bias=None, allowed=None):
    R, V = z.shape
    out, mag = z.double().clone(), z.double().abs()
    if history is not None:
        for r in range(R):
            h = history if history.dim() == 1 else history[r]
            n = len(h) if hist_len is None else max(0, min(len(h), int(hist_len[r])))
            rep, freq, pres = (penalties if penalties.dim() == 1 else penalties[r]).double().tolist()
            counts = {}
            for t in h[:n].tolist():
                if 0 <= t < V:
                    counts[t] = counts.get(t, 0) + 1
            for t, c in counts.items():
                v = out[r, t].item()
                v = v / rep if v > 0 else v * rep
                out[r, t] = v - freq * c - pres
                mag[r, t] = abs(v) + abs(freq) * c + abs(pres)
    if bias is not None:
        out, mag = out + bias.double(), mag + bias.double().abs()
    if allowed is not None:
        v = torch.arange(V, device=z.device)
        a = allowed.long()[..., v // 32] >> (v % 32) & 1
        out = torch.where((a == 1).expand_as(out), out, -math.inf)
    # at most five f32 roundings of values up to mag, then one to the type
    tol = 5 * 2.0 ** -24 * mag
    fin = torch.finfo(z.dtype)
    return out, tol + half_step(z.dtype) * (torch.nan_to_num(out.abs(), nan=0.0, posinf=0.0) + tol) + fin.smallest_normal * fin.eps


def check_logits(z, out=None, **kw):
    from edge_maskgit_b200 import runtime as rt
    ref, tol = logits_ref(z, **kw)
    y = rt.logits_adjust(z, out=out, **kw)
    assert y.dtype == z.dtype
    within(y, ref, tol)
    return y


def ints(lo, hi, *shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("R,V,L", [(1, 1, 1), (2, 7, 3), (3, 31, 40), (5, 2025, 257), (4, 4096, 100), (3, 4099, 1000),
                                   (2, 50001, 3000)])
def test_logits_all(dt, R, V, L):
    words = (V + 31) // 32
    check_logits(randn(R, V, dtype=dt, seed=20, std=3.0), history=ints(-2, max(2, V // 4) + 2, R, L, seed=21),
                 hist_len=ints(-1, L + 2, R, seed=22), penalties=torch.tensor([1.3, 0.4, 0.2], device="cuda").repeat(R, 1),
                 bias=randn(R, V, dtype=F32, seed=23), allowed=ints(-2 ** 31, 2 ** 31 - 1, R, words, seed=24))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("V", [2045, 2046, 2047, 2048, 4089, 4093, 4095, 4096, 8189, 8191, 8192])
@pytest.mark.parametrize("R", [6, 400])
def test_logits_rows_that_end_at_a_chunks_border(dt, V, R):
    """A row may fill its last chunk exactly, pass it by its lead, or leave it empty."""
    kw = dict(history=ints(-2, V + 2, R, 9, seed=81), penalties=torch.tensor([1.3, 0.4, 0.2], device="cuda"),
              bias=randn(V, dtype=F32, seed=82), allowed=ints(-2 ** 31, 2 ** 31 - 1, (V + 31) // 32, seed=83))
    z = randn(R, V, dtype=dt, seed=84, std=3.0)
    from edge_maskgit_b200 import runtime as rt
    y = rt.logits_adjust(z, **kw)
    rows = list(range(min(R, 8))) + [R - 1]
    pick = dict(kw, history=kw["history"][rows])
    within(y[rows], *logits_ref(z[rows], **pick))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hist", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mask", [False, True])
def test_logits_parts_shared_rows_in_place(dt, hist, bias, mask):
    R, V = 5, 2025
    kw = {}
    if hist:
        kw.update(history=ints(0, 300, 257, seed=25), penalties=torch.tensor([0.7, -0.4, 0.2], device="cuda"))
    if bias:
        kw.update(bias=randn(V, dtype=F32, seed=26))
    if mask:
        kw.update(allowed=ints(-2 ** 31, 2 ** 31 - 1, (V + 31) // 32, seed=27))
    z = randn(R, V, dtype=dt, seed=28, std=3.0)
    want = check_logits(z, **kw)
    again = z.clone()
    from edge_maskgit_b200 import runtime as rt
    assert rt.logits_adjust(again, out=again, **kw) is again
    assert torch.equal(again, want)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("parts", range(8))
def test_logits_many_rows_of_many_tokens(dt, parts):
    """Every combination of parts at a size where each row is cut into its longest chunks."""
    from edge_maskgit_b200 import runtime as rt
    R, V = 200, 60001
    kw = {}
    if parts & 1:
        kw.update(history=ints(0, V, R, 33, seed=36), penalties=torch.tensor([1.4, 0.3, 0.2], device="cuda"))
    if parts & 2:
        kw.update(bias=randn(V, dtype=F32, seed=37))
    if parts & 4:
        kw.update(allowed=ints(-2 ** 31, 2 ** 31 - 1, R, (V + 31) // 32, seed=38))
    z = randn(R, V, dtype=dt, seed=39, std=3.0)
    y = rt.logits_adjust(z, **kw)
    rows = [0, 1, 2, 7, 77, R - 1]
    pick = {k: (v[rows] if v.dim() == 2 else v) for k, v in kw.items()}
    within(y[rows], *logits_ref(z[rows], **pick))


@pytest.mark.parametrize("dt", [F32, F16])
def test_logits_strided_rows(dt):
    R, V = 4, 1003
    wide = randn(R, V + 9, dtype=dt, seed=29)
    for lo in range(4):
        for out_lo in (lo, 1, 4):
            out = torch.zeros(R, V + 9, dtype=dt, device="cuda")
            check_logits(wide[:, lo:lo + V], out=out[:, out_lo:out_lo + V], history=ints(0, V, R, 50, seed=30)[:, 3:40],
                         penalties=torch.tensor([2.0, 0.5, 0.25], device="cuda"), bias=randn(R, V + 3, dtype=F32, seed=31)[:, 1:1 + V],
                         allowed=ints(-2 ** 31, 2 ** 31 - 1, R, V // 32 + 4, seed=32)[:, 2:2 + (V + 31) // 32])
            assert not out[:, :out_lo].any() and not out[:, out_lo + V:].any()


def test_logits_masks_win_over_everything():
    from edge_maskgit_b200 import runtime as rt
    z = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, torch.finfo(F32).min] * 8] * 2, device="cuda")
    none = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    y = rt.logits_adjust(z, allowed=none, history=ints(0, 40, 2, 9, seed=33), penalties=torch.tensor([1.5, 1.0, 1.0], device="cuda"))
    assert (y == -math.inf).all()
    assert torch.equal(rt.logits_adjust(z, allowed=~none).nan_to_num(7.0), z.nan_to_num(7.0))
    empty = rt.logits_adjust(z, history=ints(0, 40, 2, 0, seed=34), penalties=torch.tensor([1.5, 1.0, 1.0], device="cuda"))
    assert torch.equal(empty.nan_to_num(7.0), z.nan_to_num(7.0))
    assert rt.logits_adjust(z[:0]).shape == (0, 40)


def test_logits_many_repeats():
    """One token 70000 times: counts are whole numbers of any size."""
    check_logits(randn(2, 100, dtype=F32, seed=35), history=torch.full((2, 70000), 7, dtype=torch.int32, device="cuda"),
                 penalties=torch.tensor([1.0, 0.001, 0.5], device="cuda"))


# --------------------------------------------------------------------------------- attention
def attention_ref(q, k, v, scale=None, cap=0.0, slopes=None, dist_bias=None, causal=False, prefix=None, k_len=None,
                  q_pos=None, doc_q=None, doc_k=None):
    """(out, tolerance) in 64 bits, from the formulas, one batch row and head at a time."""
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    j = torch.arange(Sk, device=q.device)[None]
    for b in range(B):
        p = (Sk - Sq if q_pos is None else int(q_pos[b])) + torch.arange(Sq, device=q.device)[:, None]
        seen = (j < (Sk if k_len is None else int(k_len[b]))).expand(Sq, Sk).clone()
        if causal:
            seen &= (j <= p) | (j < (0 if prefix is None else int(prefix[b])))
        if doc_q is not None:
            seen &= (doc_q[b][:, None] == doc_k[b][None]) & (doc_q[b][:, None] >= 0)
        for h in range(Hq):
            qq, kk, vv = q[b, :, h].double(), k[b, :, h // (Hq // Hkv)].double(), v[b, :, h // (Hq // Hkv)].double()
            any_key = seen.any(0)
            kk = torch.where(any_key[:, None], kk, 0.0)   # never looked at
            s = qq @ kk.t() * scale
            err = (D + 4) * U22 * (qq.abs() @ kk.abs().t()) * abs(scale)
            if cap:
                s = cap * torch.tanh(s / cap)
                err = err + 8 * U22 * cap
            if slopes is not None:
                s = s - slopes[h].double() * (p - j).abs()
            if dist_bias is not None:
                R = dist_bias.shape[1] // 2
                s = s + dist_bias[h].double()[(j - p).clamp(-R, R) + R]
            s = torch.where(seen, s, -math.inf)
            live = s > -math.inf
            m = s.amax(1, keepdim=True) if Sk else torch.full((Sq, 1), -math.inf, device=q.device, dtype=torch.float64)
            e = torch.where(live | s.isnan(), torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = e.sum(1, keepdim=True)
            w = e / torch.where(l == 0, 1.0, l)
            # a key that a row does not see contributes nothing, whatever v holds
            contrib = torch.where((live | s.isnan()).t()[:, :, None], w.t()[:, :, None] * vv[:, None, :], 0.0) \
                if not torch.isfinite(vv).all() else None
            out[b, :, h] = contrib.sum(0) if contrib is not None else w @ vv
            mag = torch.nan_to_num(w) @ torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0).abs()
            # score errors (rounded in base 2 up to the score's size) act on p and on the sum
            big = torch.where(live, s.abs(), 0.0).amax(1, keepdim=True) if Sk else 0.0
            e_s = torch.where(live, err, 0.0).amax(1, keepdim=True) + 4 * U22 * big + 8 * U22 if Sk else 0.0
            tol[b, :, h] = (half_step(q.dtype) + 2 * e_s + (Sk + 8) * U22) * mag
    fin = torch.finfo(q.dtype)
    tol = tol + half_step(q.dtype) * (out.abs().nan_to_num(0.0, 0.0, 0.0) + tol) + fin.smallest_normal * fin.eps
    return out, tol


def check_attention(q, k, v, out=None, **kw):
    from edge_maskgit_b200 import runtime as rt
    ref, tol = attention_ref(q, k, v, **kw)
    y = rt.attention(q, k, v, out=out, **kw)
    assert y.dtype == q.dtype and y.shape == q.shape
    within(y, ref, tol)
    return y


def qkv(B, Sq, Sk, Hq, Hkv, D, dt, seed=40):
    return (randn(B, Sq, Hq, D, dtype=dt, seed=seed), randn(B, Sk, Hkv, D, dtype=dt, seed=seed + 1),
            randn(B, Sk, Hkv, D, dtype=dt, seed=seed + 2))


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 17, 4, 2, 64), (1, 1, 1000, 8, 1, 128), (3, 5, 300, 4, 4, 48), (1, 16, 129, 2, 2, 80),
         (2, 127, 127, 2, 1, 64), (1, 128, 128, 1, 1, 128), (1, 129, 257, 3, 3, 48), (1, 257, 257, 4, 4, 48),
         (2, 300, 300, 4, 2, 128), (1, 513, 700, 2, 1, 104), (1, 700, 90, 2, 2, 32), (2, 33, 2000, 14, 2, 64),
         (1, 1, 5000, 16, 1, 40)]
# enough rows and keys for the 128-row tiles, with small and large heads
SIZES += [(40, 129, 257, 3, 3, 48), (16, 257, 257, 4, 4, 48), (10, 300, 300, 4, 2, 64), (6, 513, 700, 2, 2, 64),
          (6, 129, 1000, 4, 4, 32), (1, 1500, 1500, 3, 1, 8), (6, 129, 257, 3, 3, 128), (12, 700, 90, 2, 2, 104),
          (3, 400, 2100, 2, 2, 72), (1, 2000, 130, 8, 8, 64)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hkv,D", SIZES)
def test_attention_plain_and_causal(dt, B, Sq, Sk, Hq, Hkv, D):
    q, k, v = qkv(B, Sq, Sk, Hq, Hkv, D, dt)
    check_attention(q, k, v)
    check_attention(q, k, v, causal=True)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hkv,D", [(2, 1, 300, 4, 2, 64), (2, 5, 1100, 8, 2, 128), (2, 150, 150, 4, 4, 48),
                                              (1, 400, 650, 4, 2, 128), (2, 290, 290, 2, 2, 96),
                                              (28, 150, 150, 4, 4, 48), (5, 290, 290, 2, 2, 96), (4, 700, 900, 2, 2, 64)])
@pytest.mark.parametrize("shape", ["cap", "slopes", "table", "narrow", "all"])
def test_attention_shaped_scores(dt, B, Sq, Sk, Hq, Hkv, D, shape):
    q, k, v = qkv(B, Sq, Sk, Hq, Hkv, D, dt)
    kw = {}
    if shape in ("cap", "all"):
        kw.update(cap=5.0, scale=0.5)
    if shape in ("slopes", "all"):
        kw.update(slopes=2.0 ** -torch.arange(1.0, Hq + 1, device="cuda"))
    if shape in ("table", "all"):
        kw.update(dist_bias=randn(Hq, 2 * 200 + 1, dtype=F32, seed=50))
    if shape == "narrow":
        kw.update(dist_bias=randn(Hq, 2 * 3 + 1, dtype=F32, seed=51, std=2.0))
    check_attention(q, k, v, **kw)
    check_attention(q, k, v, causal=True, prefix=i32(*range(60, 60 + B)), **kw)


@pytest.mark.parametrize("S,D", [(40, 64), (700, 64), (700, 128)])
@pytest.mark.parametrize("cap,scale", [(2.0 ** -10, 2.0 ** 10), (2.0 ** 10, 0.125), (2.0 ** 10, 200.0), (0.0, 2.0 ** 100)])
def test_attention_constants_at_their_bounds(S, D, cap, scale):
    q, k, v = qkv(1, S, S, 4, 2, D, F16, seed=66)
    if scale > 1e3:   # scores of 0 and of one size: each is either nothing or far past the cap
        q, k = torch.zeros_like(q), torch.zeros_like(k)
        q[..., 0], k[:, S // 2:, :, 0] = 1.0, -1.0
    check_attention(q, k, v, cap=cap, scale=scale)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("S,D", [(700, 128), (1100, 48), (1300, 48)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_far_beyond_the_table(dt, S, D, cap, slopes, causal):
    """A table much narrower than the sequence: most keys take one of its two end values, which
    differ enough to matter."""
    q, k, v = qkv(1, S, S, 2, 2, D, dt)
    table = randn(2, 2 * 20 + 1, dtype=F32, seed=53)
    table[:, 0], table[:, -1] = 1.5, -1.0
    check_attention(q, k, v, cap=cap, dist_bias=table, causal=causal,
                    slopes=torch.tensor([0.002, 0.0], device="cuda") if slopes else None)


@pytest.mark.parametrize("Sq,Sk", [(1, 500), (3, 500), (200, 500), (385, 385), (300, 500), (40, 3000)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths_positions_and_empty_rows(Sq, Sk, causal):
    """Lengths of zero and one, past the end and negative; positions before the first key."""
    q, k, v = qkv(6, Sq, Sk, 4, 2, 64, BF16)
    k_len = i32(0, 1, Sk, Sk + 9, -3, Sk // 2)
    pos = i32(0, -5, Sk - Sq, 3, 7, Sk // 2 - Sq)
    y = check_attention(q, k, v, causal=causal, k_len=k_len, q_pos=pos)
    assert not y[0].any() and not y[4].any()
    if causal:
        assert not y[1, :min(Sq, 5)].any()
        check_attention(q, k, v, causal=True, k_len=k_len, q_pos=pos, prefix=i32(5, 5, 0, -1, 9, 10 ** 6))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[300], [1, 2, 3, 250, 44], [128, 128, 44], [100, 5, 170, 3], [40] * 7])
@pytest.mark.parametrize("B,D", [(2, 48), (20, 48), (6, 128)])
def test_attention_documents(dt, causal, lens, B, D):
    S = sum(lens) + 11
    ids = torch.tensor([i for i, n in enumerate(lens) for _ in range(n)] + [-1] * 11, dtype=torch.int32, device="cuda")
    q, k, v = qkv(B, S, S, 4, 2, D, dt)
    doc = torch.stack([ids, ids.flip(0)]).repeat(B // 2, 1).contiguous()
    y = check_attention(q, k, v, causal=causal, doc_q=doc, doc_k=doc, dist_bias=randn(4, 101, dtype=F32, seed=52))
    assert not y[0, -11:].any() and not y[1, :11].any()
    # a document's rows are what it gives alone
    n = lens[0]
    alone = check_attention(q[:1, :n], k[:1, :n], v[:1, :n], causal=causal, dist_bias=randn(4, 101, dtype=F32, seed=52))
    assert (alone - y[:1, :n]).abs().max() <= 4 * half_step(dt) * max(1.0, v.abs().max().item())


def test_attention_documents_in_any_order():
    g = torch.Generator(device="cuda").manual_seed(3)
    for Sq, Sk in ((1, 300), (9, 200), (330, 330), (1000, 1000), (600, 1500)):
        dq = torch.randint(-1, 4, (2, Sq), generator=g, device="cuda", dtype=torch.int32)
        dk = torch.randint(-1, 5, (2, Sk), generator=g, device="cuda", dtype=torch.int32)
        q, k, v = qkv(2, Sq, Sk, 2, 2, 64, F16)
        check_attention(q, k, v, doc_q=dq, doc_k=dk)
        check_attention(q, k, v, doc_q=dq, doc_k=dk, causal=True, prefix=i32(70, 0), k_len=i32(Sk, Sk - 40))


@pytest.mark.parametrize("Sq,Sk,D", [(1, 260, 64), (4, 700, 64), (260, 260, 64), (420, 420, 128), (900, 900, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_unseen_keys_may_hold_anything(Sq, Sk, D, bad):
    """NaN and infinities behind k_len, in another document, and after a causal row's position."""
    q, k, v = qkv(2, Sq, Sk, 2, 1, D, F16)
    k_len = i32(Sk - 37, Sk)
    k[0, Sk - 37:], v[0, Sk - 37:] = bad, bad
    y = check_attention(q, k, v, k_len=k_len)
    assert y[0].isfinite().all()
    doc_k = torch.zeros(2, Sk, dtype=torch.int32, device="cuda")
    doc_q = torch.zeros(2, Sq, dtype=torch.int32, device="cuda")
    doc_k[:, 20:30] = 1
    k[:, 20:30], v[:, 20:30] = bad, bad
    check_attention(q, k, v, k_len=k_len, doc_q=doc_q, doc_k=doc_k)
    if Sq == Sk:   # keys after a row's own position
        q, k, v = qkv(2, Sq, Sk, 2, 1, D, F16)
        v[0, 100:] = bad
        y = check_attention(q, k, v, causal=True)
        assert y[0, :100].isfinite().all() and not y[0, 100:].isfinite().any() and y[1].isfinite().all()
        q, k, v = qkv(2, Sq, Sk, 2, 1, D, F16)   # a NaN score that is seen makes its rows NaN, no others
        k[1, 150, 0] = math.nan
        y = check_attention(q, k, v, causal=True)
        assert y[1, :150].isfinite().all() and y[1, 150:].isnan().all() and y[0].isfinite().all()


@pytest.mark.parametrize("Sq,Sk", [(1, 300), (290, 290), (1300, 1300)])
def test_attention_lowest_values_and_hidden_distances(Sq, Sk):
    low = torch.finfo(F32).min
    q, k, v = qkv(1, Sq, Sk, 2, 2, 64, BF16)
    table = torch.zeros(2, 2 * 300 + 1, device="cuda")
    table[0] = low          # the lowest value everywhere: a uniform row, not an empty one
    table[1] = -math.inf    # all hidden: an empty row
    y = check_attention(q, k, v, dist_bias=table)
    assert y[:, :, 0].any() and not y[:, :, 1].any()
    table[:] = -math.inf    # a window by distance
    table[:, 300 - 20:300 + 1] = 0.5
    check_attention(q, k, v, dist_bias=table)
    table[:] = low
    table[:, 300 - 20:300 + 1] = 0.5
    check_attention(q, k, v, dist_bias=table)


@pytest.mark.parametrize("Sq,Sk", [(2, 300), (260, 260), (1300, 1300)])
def test_attention_large_scores(Sq, Sk):
    q, k, v = qkv(1, Sq, Sk, 2, 2, 64, BF16)
    check_attention(q * 30, k * 30, v, scale=1.0)
    check_attention(q * 30, k * 30, v, scale=1.0, cap=50.0)
    check_attention(q, k, v, scale=-2.0)
    check_attention(q, k, v, scale=0.0)


@pytest.mark.parametrize("S,Hq,Hkv,D", [(1, 4, 4, 48), (40, 8, 2, 64), (300, 4, 2, 128)])
def test_attention_strides(S, Hq, Hkv, D):
    """q | k | v of one projection, heads-first tensors, a shared cache, rows of a wider output."""
    packed = randn(2, S, Hq + 2 * Hkv, D, dtype=F16, seed=60)
    q, k, v = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], packed[:, :, Hq + Hkv:]
    wide = torch.zeros(2, S + 2, Hq, D + 8, dtype=F16, device="cuda")
    check_attention(q, k, v, causal=True, out=wide[:, 1:S + 1, :, 8:])
    assert not wide[:, 0].any() and not wide[:, S + 1].any() and not wide[..., :8].any()
    kh, vh = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    check_attention(q, kh, vh)
    check_attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1))
    check_attention(q, k[:, :, :1].expand(-1, -1, Hkv, -1), v)
    check_attention(q, k[:, :1].expand(-1, S, -1, -1), v, causal=True)


def test_attention_no_keys_and_no_rows():
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(2, 3, 4, 2, 2, 64, F16)
    assert not rt.attention(q, k[:, :0], v[:, :0]).any()
    assert rt.attention(q[:, :0], k, v).shape == (2, 0, 2, 64)
    assert rt.attention(q[:0], k[:0], v[:0]).shape == (0, 3, 2, 64)


def test_attention_long_cache_offsets():
    """A cache of more than 2^31 elements: offsets past 32 bits."""
    S = 70001
    cache = torch.zeros(4, S, 64, 128, dtype=F16, device="cuda")   # 2.3e9 elements
    k = cache.normal_(generator=torch.Generator(device="cuda").manual_seed(5))[:, :, :32]
    v = cache[:, :, 32:]
    q = randn(4, 1, 32, 128, dtype=F16, seed=61)
    ref, tol = attention_ref(q[3:, :, 30:], k[3:, :, 30:], v[3:, :, 30:])
    from edge_maskgit_b200 import runtime as rt
    within(rt.attention(q, k, v)[3:, :, 30:], ref, tol)
    q = randn(4, 200, 32, 128, dtype=F16, seed=62)
    ref, tol = attention_ref(q[3:, :, 31:], k[3:, :, 31:], v[3:, :, 31:], causal=True)
    within(rt.attention(q, k, v, causal=True)[3:, :, 31:], ref, tol)


# ------------------------------------------------------------------------------ streams, graphs
def _step(x, st):
    """A 16-bit transformer step: projection, attention, output layer, MLP, logits, adjustment."""
    from edge_maskgit_b200 import runtime as rt
    B, S, H, D = st["B"], st["S"], 4, 48
    qkv_ = rt.linear(x, st["wqkv"], bias=st["bqkv"]).view(B, S, 3, H, D)
    a = rt.attention(*qkv_.unbind(2), dist_bias=st["table"], doc_q=st["doc"], doc_k=st["doc"], cap=20.0)
    x = rt.linear(a.view(B * S, H * D), st["wo"], resid=x)
    u = rt.linear(x, st["wu"], bias=st["bu"], act=1)
    x = rt.linear(u, st["wd"], resid=x)
    z = rt.linear(x, st["head"])
    return rt.logits_adjust(z, history=st["hist"], penalties=st["pen"], allowed=st["allowed"])


def _step_state(B=2, S=150, V=515, dt=BF16):
    E, F = 192, 512
    w = lambda n, k, s: randn(n, k, dtype=dt, seed=s, std=k ** -0.5)  # noqa: E731
    doc = torch.arange(S, device="cuda", dtype=torch.int32).div(64, rounding_mode="floor").int().expand(B, S).contiguous()
    return dict(B=B, S=S, wqkv=w(3 * E, E, 70), bqkv=randn(3 * E, dtype=F32, seed=71, std=0.1), wo=w(E, E, 72), wu=w(F, E, 73),
                bu=randn(F, dtype=F32, seed=74, std=0.1), wd=w(E, F, 75), head=w(V, E, 76), table=randn(4, 65, dtype=F32, seed=77),
                doc=doc, hist=ints(0, V, 40, seed=78), pen=torch.tensor([1.2, 0.1, 0.2], device="cuda"),
                allowed=ints(-2 ** 31, 2 ** 31 - 1, (V + 31) // 32, seed=79)), randn(B * S, E, dtype=dt, seed=80)


def _step_ref(x, st):
    """The same step, each operator from the GPU operator's own input type, in 64 bits between roundings."""
    dt, B, S = x.dtype, st["B"], st["S"]
    r = lambda t: t.to(dt)  # noqa: E731
    qkv_ = r(linear_ref(x, st["wqkv"], st["bqkv"], 0, None)[0]).view(B, S, 3, 4, 48)
    a = r(attention_ref(*qkv_.unbind(2), dist_bias=st["table"], doc_q=st["doc"], doc_k=st["doc"], cap=20.0)[0])
    x = r(linear_ref(a.view(B * S, -1), st["wo"], None, 0, x)[0])
    u = r(linear_ref(x, st["wu"], st["bu"], 1, None)[0])
    x = r(linear_ref(u, st["wd"], None, 0, x)[0])
    z = r(linear_ref(x, st["head"], None, 0, None)[0])
    return logits_ref(z, history=st["hist"], penalties=st["pen"], allowed=st["allowed"])[0]


@pytest.mark.parametrize("B", [2, 30])
def test_a_step_of_all_three(B):
    """Six roundings to bf16 follow one another, each of relative size 2^-8 at most and spread over
    sums: the 2-norm of the difference stays below their plain sum, 6 * 2^-8 of the result's."""
    st, x = _step_state(B)
    y, ref = _step(x, st), _step_ref(x, st)
    live = ref > -math.inf
    assert torch.equal(live, y > -math.inf)
    assert ((y.double() - ref)[live].norm() / ref[live].norm()).item() < 6 * 2.0 ** -8


@pytest.mark.parametrize("B", [2, 30])
def test_streams_and_graph_replays_agree(B):
    st, x = _step_state(B)
    want = _step(x, st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _step(x, st)
    side.synchronize()
    assert torch.equal(want, other)
    graphs = []
    for shift in (0.0, 1.0):   # two graphs, replayed at the same time on two streams
        buf = x + shift
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(buf, st)
        graphs.append((g, buf, out, _step(x + shift, st)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, buf, out, ref in graphs:
        assert torch.equal(out, ref)


def test_split_attention_in_two_graphs():
    """The decode form's workspace belongs to its call: two captured calls do not share one."""
    from edge_maskgit_b200 import runtime as rt
    calls = []
    for seed in (90, 95):
        q, k, v = qkv(2, 1, 3000, 8, 2, 64, F16, seed=seed)
        want = rt.attention(q, k, v)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = rt.attention(q, k, v)
        calls.append((g, out, want, (q, k, v)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, *_), s in zip(calls, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, out, want, _ in calls:
        assert torch.equal(out, want)


def test_gpu_refusals():
    from edge_maskgit_b200 import runtime as rt
    x, w = randn(4, 64, dtype=F16, seed=1), randn(8, 64, dtype=F16, seed=2)
    for bad in (lambda: rt.linear(x, w.bfloat16()), lambda: rt.linear(x, w[:, :56]), lambda: rt.linear(x[:, :60], w[:, :60]),
                lambda: rt.linear(x.t(), w), lambda: rt.linear(x, w, bias=randn(8, dtype=F16, seed=3)),
                lambda: rt.linear(x, w, bias=randn(7, dtype=F32, seed=3)), lambda: rt.linear(x, w, act=5),
                lambda: rt.linear(x, w, resid=x), lambda: rt.linear(x, w.cpu()), lambda: rt.linear(x, w, out=torch.empty(4, 8, device="cuda")),
                lambda: rt.linear(x, w.clone().requires_grad_()), lambda: rt.linear(x[:, 4:60], w[:, :56])):
        with pytest.raises(rt.MgcError):
            bad()
    q, k, v = qkv(2, 3, 5, 4, 2, 64, F16)
    for bad in (lambda: rt.attention(q, k, v[:, :4]), lambda: rt.attention(q[:, :, :3], k, v), lambda: rt.attention(q, k, v.bfloat16()),
                lambda: rt.attention(q[..., :60], k[..., :60], v[..., :60]), lambda: rt.attention(q, k, v, prefix=i32(1, 1)),
                lambda: rt.attention(q, k, v, k_len=i32(1)), lambda: rt.attention(q, k, v, doc_q=ints(0, 2, 2, 3, seed=1)),
                lambda: rt.attention(q, k, v, slopes=torch.ones(2, device="cuda")), lambda: rt.attention(q, k, v, cap=-1.0),
                lambda: rt.attention(q, k, v, dist_bias=torch.ones(4, 4, device="cuda")), lambda: rt.attention(q, k, v, scale=math.inf),
                lambda: rt.attention(q.transpose(2, 3), k, v), lambda: rt.attention(q, k, v, out=torch.empty_like(q)[:, :2])):
        with pytest.raises(rt.MgcError):
            bad()
    z = randn(3, 40, dtype=F32, seed=4)
    h, pen = ints(0, 9, 3, 5, seed=5), torch.ones(3, 3, device="cuda")
    for bad in (lambda: rt.logits_adjust(z, history=h), lambda: rt.logits_adjust(z, penalties=pen), lambda: rt.logits_adjust(z.t()),
                lambda: rt.logits_adjust(z, bias=torch.ones(39, device="cuda")), lambda: rt.logits_adjust(z, hist_len=i32(1, 1, 1)),
                lambda: rt.logits_adjust(z, allowed=ints(0, 2, 3, seed=6)), lambda: rt.logits_adjust(z, history=h.long(), penalties=pen),
                lambda: rt.logits_adjust(z, history=h[:2], penalties=pen), lambda: rt.logits_adjust(z, out=torch.empty(3, 40, device="cuda", dtype=F16))):
        with pytest.raises(rt.MgcError):
            bad()
