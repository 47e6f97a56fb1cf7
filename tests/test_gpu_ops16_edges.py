"""GPU: the 16-bit operators where they can go wrong at the ends of their ranges: the lowest bias, values near
the largest, probabilities far below a row's maximum, padding documents, far positions, workspaces.

Tolerances as in test_gpu_ops16: half a step for each rounding (probabilities, result) and n 2^-22 for sums of
n terms, here with the size of a score taken over the keys whose weight is not 0."""
import math

import pytest

from test_gpu_ops16 import BF16, F16, F32, U22, attention_ref, half_step, i32, ints, qkv, randn, within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield torch.device("cuda:0")
    from edge_maskgit_b200 import runtime as rt
    torch.cuda.synchronize()
    assert rt.device_error() == 0


def scores_ref(q, k, v, bias, seen, scale=None):
    """(out, tolerance) in 64 bits of softmax(scale q.k + bias) v over the seen keys; bias and seen [Hq][Sq][Sk], equal heads."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    Sk, fin = k.shape[1], torch.finfo(q.dtype)
    qq, kk, vv = (t[0].double().transpose(0, 1) for t in (q, k, v))
    s = torch.where(seen, qq @ kk.mT * scale + bias, -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    w = w / torch.where(m == -math.inf, 1.0, w.sum(-1, keepdim=True))
    out, mag = w @ vv, w @ vv.abs()
    err = (q.shape[-1] + 4) * U22 * (qq.abs() @ kk.abs().mT) * abs(scale) + 4 * U22 * s.abs()
    # (a score that its bias absorbs is the bias itself, here and in 32 bits: no error)
    e_s = torch.where((w > 0) & (s != bias), err, 0.0).amax(-1, keepdim=True) + 8 * U22
    tol = (half_step(q.dtype) + 2 * e_s + (Sk + 8) * U22) * mag
    tol = tol + half_step(q.dtype) * (out.abs() + tol) + fin.smallest_normal * fin.eps
    return out.transpose(0, 1)[None], tol.transpose(0, 1)[None]


# ---------------------------------------------------------------------------- lowest biases
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,reach", [(1, 300, 40), (40, 300, 40), (700, 700, 100), (1300, 1300, 300), (300, 2000, 1)])
@pytest.mark.parametrize("slopes", [False, True])
def test_attention_lowest_bias_everywhere(dt, D, Sq, Sk, reach, slopes):
    """Every score is absorbed by the lowest bias: a uniform row, however large the scores are, in tiles whose
    distances lie inside the table and in those beyond it."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 2, 2, D, dt)
    table = torch.full((2, 2 * reach + 1), torch.finfo(F32).min, device="cuda")
    for causal in (False, True):
        seen = torch.ones(Sq, Sk, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(Sk - Sq)
        y = rt.attention(q, k, v, scale=4.0, dist_bias=table, causal=causal,
                         slopes=torch.tensor([0.01, 0.0], device="cuda") if slopes else None)
        within(y, *scores_ref(q, k, v, torch.finfo(F32).min, seen, scale=4.0))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk", [(1, 300), (40, 300), (700, 700), (1300, 1300)])
def test_attention_lowest_bias_as_a_window(dt, D, Sq, Sk):
    """The lowest value outside a window of distances: it hides a key wherever another is inside."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 2, 2, D, dt)
    reach = 300
    table = torch.full((2, 2 * reach + 1), torch.finfo(F32).min, device="cuda")
    table[0, reach - 20:reach + 1] = 0.5
    table[1, reach + 250:] = -0.5   # far keys only: rows near the end see lowest biases alone
    j, p = torch.arange(Sk, device="cuda")[None], Sk - Sq + torch.arange(Sq, device="cuda")[:, None]
    bias = table.double()[:, (j - p).clamp(-reach, reach) + reach]
    y = rt.attention(q, k, v, scale=3.0, dist_bias=table)
    within(y, *scores_ref(q, k, v, bias, torch.ones_like(bias, dtype=torch.bool), scale=3.0))


# --------------------------------------------------------------------- values near the largest
@pytest.mark.parametrize("Sq,Sk", [(1, 5), (1, 300), (1, 9000), (3, 700), (40, 300), (300, 300), (700, 3000), (64, 9000)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_values_near_the_largest(Sq, Sk, D, causal):
    """Averages of values up to 2^127.9 are finite, also where their sum is not."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 4, 2, D, BF16)
    unit = 1.0 + v.float().abs().clamp(max=2.9) * 0.33   # 1 .. 1.957
    sign = torch.ones(2, device="cuda")
    sign[1] = -1.0
    small = (unit * sign[None, None, :, None]).to(BF16)
    ref, tol = attention_ref(q, k, small, causal=causal, scale=0.5)
    y = rt.attention(q, k, (small.float() * 2.0 ** 127).to(BF16), causal=causal, scale=0.5)
    within(y.double() * 2.0 ** -127, ref, tol)


# ------------------------------------------------------------- probabilities far below the maximum
@pytest.mark.parametrize("Sq,Sk", [(1, 300), (1, 3000), (1, 16385), (40, 300), (40, 16385), (300, 5000)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gap", [13.0, 14.0, 15.0, 16.0, 17.0])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_attention_many_keys_far_below_one(Sq, Sk, D, gap, where):
    """One key takes the row's weight and has a value of 0: what is left is the many keys 13 to 17 below it."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 2, 2, D, F16)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    v = v.abs() + 0.5
    at = {"first": 0, "middle": Sk // 2, "last": Sk - 1}[where]
    q[..., 0], k[:, at, :, 0], v[:, at] = 1.0, gap, 0.0
    ref, tol = attention_ref(q, k, v, scale=1.0)
    within(rt.attention(q, k, v, scale=1.0), ref, tol)


# ------------------------------------------------------------------------------- documents
@pytest.mark.parametrize("Sq,Sk,D", [(1, 300, 64), (40, 300, 64), (900, 900, 64), (900, 900, 128), (600, 1500, 48)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_padding_of_any_negative_number(Sq, Sk, D, causal):
    """A query with a negative document number sees nothing, whatever negative numbers the keys have."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(2, Sq, Sk, 2, 2, D, F16)
    dq, dk = ints(-4, 3, 2, Sq, seed=100), ints(-4, 3, 2, Sk, seed=101)
    y = rt.attention(q, k, v, doc_q=dq, doc_k=dk, causal=causal)
    assert not y[dq < 0].any()
    within(y, *attention_ref(q, k, v, doc_q=dq, doc_k=dk, causal=causal))


# ---------------------------------------------------------------------------- far positions
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 300, 64), (1, 9000, 128), (40, 300, 64), (700, 700, 64), (700, 700, 128)])
@pytest.mark.parametrize("far", [10 ** 5, 10 ** 6, 2 ** 29 - 10 ** 4, -10 ** 6])
def test_attention_slopes_of_far_positions(dt, Sq, Sk, D, far):
    """Slopes fall off by distance, however far the first key is: a constant of the row takes no part."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 2, 2, D, dt)
    slopes = torch.tensor([0.4, 0.01], device="cuda")
    p = far + torch.arange(Sq, device="cuda")[:, None]
    j = torch.arange(Sk, device="cuda")[None]
    near = -slopes.double()[:, None, None] * ((p - j).abs() - (p - p.clamp(0, Sk - 1)).abs())   # less the row's constant
    ref, tol = scores_ref(q, k, v, near, torch.ones_like(near, dtype=torch.bool))
    within(rt.attention(q, k, v, slopes=slopes, q_pos=i32(far)), ref, tol)


# -------------------------------------------------------------------------------- workspaces
def workspace(q, k, **kw):
    """Bytes that a call of these shapes asks for."""
    import ctypes as C
    from edge_maskgit_b200._lib import AttentionArgs, lib
    B, Sq, Hq, D = q.shape
    a = AttentionArgs(dtype=1 if q.dtype == F16 else 30, B=B, Sq=Sq, Sk=k.shape[1], Hq=Hq, Hkv=k.shape[2], D=D, scale=1.0, **kw)
    a.q_stride[:] = a.out_stride[:] = q.stride()[:3]
    a.k_stride[:] = a.v_stride[:] = k.stride()[:3]
    need = C.c_uint64()
    assert lib.mgc_attention_workspace(C.byref(a), C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hkv,D", [(2, 1, 9000, 8, 2, 64), (1, 4, 20000, 4, 1, 128), (1, 128, 4000, 2, 2, 64),
                                              (1, 200, 3000, 4, 2, 128)])
def test_attention_workspaces_of_calls_that_overlap(B, Sq, Sk, Hq, Hkv, D):
    """Partial results belong to their call: captured calls that are replayed at the same time do not share them."""
    from edge_maskgit_b200 import runtime as rt
    calls = []
    for seed in (90, 95, 99):
        q, k, v = qkv(B, Sq, Sk, Hq, Hkv, D, F16, seed=seed)
        assert workspace(q, k) >= B * Sq * Hq * 2 * (4 * D + 8)   # two ranges of keys or more
        want = rt.attention(q, k, v)
        within(want, *attention_ref(q, k, v))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = rt.attention(q, k, v)
        calls.append((g, out, want, (q, k, v)))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, *_), s in zip(calls, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, out, want, _ in calls:
        assert torch.equal(out, want)
    # the same without graphs, calls of one after another on three streams
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):
        for (_, _, want, qkv_), s in zip(calls, streams):
            with torch.cuda.stream(s):
                outs.append((rt.attention(*qkv_), want))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y, want in outs)


# ------------------------------------------------------------------------------ long caches
@pytest.mark.parametrize("B,Hkv,Sk", [(2, 1, 400000), (2, 2, 262144), (3, 1, 150000), (1, 1, 400000)])
def test_attention_long_caches_of_few_heads_fill_the_gpu(B, Hkv, Sk):
    """A long cache is cut into as many ranges of keys as there are multiprocessors, and more than 32 of them join."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(B, 1, Sk, 4 * Hkv, Hkv, 128, BF16)
    ranges = workspace(q, k) // (B * 4 * Hkv * (4 * 128 + 8))
    assert ranges * B * Hkv >= torch.cuda.get_device_properties(0).multi_processor_count
    y = rt.attention(q, k, v, k_len=i32(*[Sk - 1000 * b for b in range(B)]))
    within(y, *attention_ref(q, k, v, k_len=i32(*[Sk - 1000 * b for b in range(B)])))


# ------------------------------------------------------------------------------------- GELU
@pytest.mark.parametrize("M,N", [(1, 64), (300, 2025), (2048, 2304), (4100, 2025)])
def test_linear_gelu_keeps_small_results(M, N):
    """Sums from -13 to 0 that are exact: results down to 2^-123, relative to themselves.  The exponent of the
    Gaussian, up to 122 in base 2, takes three roundings of 2^-24 (1.6e-5 of the result at most); the rest a few 1e-6."""
    from edge_maskgit_b200 import runtime as rt
    x, w = torch.zeros(M, 8, device="cuda", dtype=BF16), torch.zeros(N, 8, device="cuda", dtype=BF16)
    w[:, 0] = -torch.linspace(0.0, 13.0, N, device="cuda").to(BF16)
    x[:, 0] = 1.0
    y = rt.linear(x, w, act=1)
    s = w[:, 0].double().expand(M, N)
    ref = s * 0.5 * torch.erfc(-s * math.sqrt(0.5))
    within(y, ref, (half_step(BF16) + 2e-5) * ref.abs())


# -------------------------------------------------------------------------------- large scores
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 200, 64), (40, 200, 64), (200, 200, 64), (2000, 200, 64), (2000, 200, 128), (400, 250, 128)])
@pytest.mark.parametrize("scale", [2.0 ** 10, -2.0 ** 16, 2.0 ** 21, 2.0 ** 28, 2.0 ** 60])
@pytest.mark.parametrize("shape", ["plain", "causal", "table", "slopes"])
def test_attention_very_large_scores(dt, Sq, Sk, D, scale, shape):
    """Scores that differ by 2^10 and more: each row is the value of its largest seen score."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 4, 4, D, dt)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    order = torch.randperm(Sk, generator=torch.Generator().manual_seed(7)).cuda()
    q[..., 0], k[..., 0] = 1.0, (order - Sk // 3).to(dt)[None, :, None]   # whole numbers below 256: exact in bf16
    kw = {"causal": dict(causal=True), "table": dict(dist_bias=randn(4, 41, dtype=F32, seed=5)),
          "slopes": dict(slopes=torch.tensor([0.5, 0.1, 0.01, 0.0], device="cuda"))}.get(shape, {})
    s = (order - Sk // 3).double() * scale
    p = Sk - Sq + torch.arange(Sq, device="cuda")[:, None]
    seen = torch.arange(Sk, device="cuda")[None] <= p if shape == "causal" else torch.ones(Sq, Sk, dtype=torch.bool, device="cuda")
    best = torch.where(seen, s, -math.inf).argmax(1)
    want = torch.where(seen.any(1)[:, None, None], v[0, best], 0.0)
    y = rt.attention(q, k, v, scale=scale, **kw)
    # two roundings: the one probability p of the row, relative to the sum's unrounded p, and the result:
    # (1 + eps / 2)^2 - 1, and the sums' few 2^-22
    h = half_step(dt)
    within(y, want.double()[None], (2 * h + h * h + 8 * U22) * want.double().abs()[None])


# ------------------------------------------------------------------------- waits that give up
@pytest.mark.parametrize("S,B,documents", [(700, 3, False), (700, 3, True), (1300, 1, False), (1300, 1, True)])
def test_attention_ends_when_a_wait_gives_up(S, B, documents):
    """One warp leaves at its second key tile as if its wait had run out: the others, which would meet it at the
    next bias window, end too, the error is reported and later calls are right."""
    import ctypes as C
    from edge_maskgit_b200 import runtime as rt
    from edge_maskgit_b200._lib import AttentionArgs, lib
    q, k, v = qkv(B, S, S, 4, 4, 64, F16)
    kw = dict(dist_bias=randn(4, 2 * 200 + 1, dtype=F32, seed=110))
    if documents:
        kw["doc_q"] = kw["doc_k"] = torch.arange(S, device="cuda", dtype=torch.int32).div(300, rounding_mode="floor").int().repeat(B, 1)
    want = rt.attention(q, k, v, **kw)
    out = torch.empty_like(q)
    a = AttentionArgs(dtype=1, B=B, Sq=S, Sk=S, Hq=4, Hkv=4, D=64, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                      out=out.data_ptr(), scale=0.125, dist_range=200, **{n: t.data_ptr() for n, t in kw.items()})
    a.q_stride[:] = a.k_stride[:] = a.v_stride[:] = a.out_stride[:] = q.stride()[:3]
    need = C.c_uint64()
    assert lib.mgc_attention_workspace(C.byref(a), C.byref(need)) == 0
    ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    torch.cuda.synchronize()
    assert lib.mgc_selftest_attention_gives_up(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert rt.device_error() == 58
    assert torch.equal(rt.attention(q, k, v, **kw), want)
    torch.cuda.synchronize()
    assert rt.device_error() == 0


# ------------------------------------------------------------------------ the rules' borders
@pytest.mark.parametrize("B,Sk,Hq,Hkv,D", [(1, 4096, 8, 2, 128), (1, 4097, 8, 2, 128), (1, 6826, 4, 1, 64), (2, 6827, 4, 1, 64),
                                           (1, 13653, 4, 4, 16), (1, 13654, 4, 4, 16), (1, 16384, 9, 9, 8), (1, 5000, 10, 10, 48)])
@pytest.mark.parametrize("Sq", [1, 3])
def test_attention_steps_on_both_sides_of_a_cluster(B, Sq, Sk, Hq, Hkv, D):
    """Key ranges that join inside a cluster, and those that join through the workspace."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(B, Sq, Sk, Hq, Hkv, D, F16)
    kw = dict(k_len=i32(*[Sk - 700 * b for b in range(B)]), causal=True)
    within(rt.attention(q, k, v, **kw), *attention_ref(q, k, v, **kw))


# --------------------------------------------------------------------------- beyond the types
def test_python_forms_refuse_what_the_c_types_cannot_hold():
    """Sizes of 2^31 and more (rows that repeat, so that they need no memory), constants beyond float32."""
    from edge_maskgit_b200 import runtime as rt
    many = 2 ** 32 + 1   # its low 32 bits are 1
    x, w = randn(1, 64, dtype=F16, seed=1), randn(8, 64, dtype=F16, seed=2)
    y = torch.zeros(1, 8, dtype=F16, device="cuda")
    z = randn(1, 8, dtype=F32, seed=3)
    h, pen = ints(0, 8, 1, seed=4), torch.ones(3, device="cuda")
    q, k, v = qkv(1, 3, 5, 2, 2, 64, F16)
    for bad in (lambda: rt.linear(x.expand(many, 64), w, out=y.expand(many, 8)),
                lambda: rt.linear(x, w[:1].expand(many, 64), out=y[:, :1].expand(1, many)),
                lambda: rt.logits_adjust(z.expand(many, 8), out=z.clone().expand(many, 8)),
                lambda: rt.logits_adjust(z, history=h.expand(many), penalties=pen),
                lambda: rt.attention(q, k[:, :1].expand(1, many, 2, 64), v[:, :1].expand(1, many, 2, 64)),
                lambda: rt.attention(q, k, v, scale=1e300), lambda: rt.attention(q, k, v, scale=-1e39),
                lambda: rt.attention(q, k, v, cap=1e39), lambda: rt.attention(q, k, v, scale=math.nan)):
        with pytest.raises(rt.MgcError):
            bad()
    assert not y.any()


# -------------------------------------------------------------------------- slopes with a table
@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("S,k_len,pos", [(40, 40, 0), (462, 462, 0), (462, 300, 100), (700, 500, 400), (922, 922, -300), (922, 600, 10 ** 5),
                                         (922, 130, 5000), (1300, 1290, -10 ** 4)])
@pytest.mark.parametrize("reach", [0, 1, 5, 40, 300])
@pytest.mark.parametrize("slope", [0.3, 30.0, 3e5])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_slopes_with_a_table(dt, D, S, k_len, pos, reach, slope, causal):
    """Both biases by distance, where the table's counts from the query and the slopes' from the nearest key."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, S, S, 2, 2, D, dt)
    table = randn(2, 2 * reach + 1, dtype=F32, seed=120)
    slopes = torch.tensor([slope, slope / 64], device="cuda")
    p, j = pos + torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None]
    bias = table.double()[:, (j - p).clamp(-reach, reach) + reach]
    bias = bias - slopes.double()[:, None, None] * ((p - j).abs() - (p - p.clamp(0, k_len - 1)).abs())
    seen = (j < k_len).expand(S, S)
    if causal:
        seen = seen & (j <= p)
    y = rt.attention(q, k, v, slopes=slopes, dist_bias=table, k_len=i32(k_len), q_pos=i32(pos), causal=causal)
    within(y, *scores_ref(q, k, v, bias, seen.expand(2, S, S)))


# ------------------------------------------------------------------------ biases of any size
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 900, 64), (40, 300, 64), (700, 700, 64), (700, 900, 128)])
@pytest.mark.parametrize("bias", [1e5, 1e7, 5e7, 9e7, 1.2e8, 1.5e8, 1.8e8, 3e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_attention_common_biases_of_any_size(dt, Sq, Sk, D, bias, sign, cap):
    """One bias for all keys takes bits of the scores, down to a uniform row, but a result stays an average."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 2, 2, D, dt)
    y = rt.attention(q, k, v, scale=2.0, cap=cap, dist_bias=torch.full((2, 1), sign * bias, device="cuda"))
    top, low = v.double().amax(1, keepdim=True), v.double().amin(1, keepdim=True)
    slack = 4 * half_step(dt) * v.double().abs().amax(1, keepdim=True)
    assert y.isfinite().all() and (y.double() <= top + slack).all() and (y.double() >= low - slack).all()
    if bias >= 1e12:
        mean, mag = v.double().mean(1, keepdim=True), v.double().abs().mean(1, keepdim=True)
        within(y, mean.expand_as(y), (half_step(dt) * (mean.abs() + mag) + (Sk + 8) * U22 * mag + 2.0 ** -24).expand_as(y))


# --------------------------------------------------------------------------------- SiLU
@pytest.mark.parametrize("M,N", [(1, 64), (300, 2025), (2048, 2304), (4100, 2025)])
def test_linear_silu_keeps_small_results(M, N):
    """Sums from -90 to 0 that are exact: results down to 2^-123, relative to themselves.  The exponential's exponent, up to
    130 in base 2, takes two roundings of 2^-24 (1.1e-5 of the result at most); the rest a few 1e-6."""
    from edge_maskgit_b200 import runtime as rt
    x, w = torch.zeros(M, 8, device="cuda", dtype=BF16), torch.zeros(N, 8, device="cuda", dtype=BF16)
    w[:, 0] = -torch.linspace(0.0, 90.0, N, device="cuda").to(BF16)
    x[:, 0] = 1.0
    y = rt.linear(x, w, act=2)
    s = w[:, 0].double().expand(M, N)
    ref = s * torch.sigmoid(s)
    within(y, ref, (half_step(BF16) + 2e-5) * ref.abs())


# ------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 300, 64), (1, 9000, 128), (3, 700, 48), (40, 300, 64), (500, 500, 64), (500, 700, 128), (128, 4000, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_one_bad_dim_leaves_the_others(dt, Sq, Sk, D, bad):
    """A NaN or infinity in one dim of a seen key's v: that dim is it, every other bit is as without it."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, Sq, Sk, 4, 2, D, dt)
    p = Sk - Sq + torch.arange(Sq, device="cuda")
    for at in (0, Sk // 3, Sk - 1):
        want = rt.attention(q, k, v, causal=True)
        w = v.clone()
        w[0, at, 1, 5] = bad
        y = rt.attention(q, k, w, causal=True)
        sees = p >= at
        hit = y[0, sees][:, 2:, 5]
        assert hit.isnan().all() if math.isnan(bad) else (hit == bad).all()
        want[0, sees.nonzero()[:, 0][:, None], torch.arange(2, 4, device="cuda")[None], 5] = 0.0
        y[0, sees.nonzero()[:, 0][:, None], torch.arange(2, 4, device="cuda")[None], 5] = 0.0
        # rows that do not see it, in a tile that holds it, have that one dim computed in another order
        near = 2 * half_step(dt) * v.abs().max().item()
        assert (y[..., 5] - want[..., 5]).abs().max().item() <= near
        y[..., 5] = want[..., 5] = 0.0
        assert torch.equal(y, want)


def test_attention_infinities_of_small_weight_and_of_both_signs():
    from edge_maskgit_b200 import runtime as rt
    for Sq, Sk, D, dt in ((1, 400, 64, F16), (300, 400, 64, F16), (300, 400, 128, BF16), (1, 9000, 64, BF16)):
        q, k, v = qkv(1, Sq, Sk, 2, 2, D, dt)
        q, k = torch.zeros_like(q), torch.zeros_like(k)
        q[..., 0], k[:, 7, :, 0] = 1.0, 100.0   # key 7 has all but e^-100 of the weight
        v[0, 9, 0, 3], v[0, 9, 1, 3], v[0, 11, 1, 3], v[0, 9, 1, 4] = math.inf, math.inf, -math.inf, -math.inf
        y = rt.attention(q, k, v, scale=1.0)
        assert (y[:, :, 0, 3] == math.inf).all() and y[:, :, 1, 3].isnan().all() and (y[:, :, 1, 4] == -math.inf).all()
        assert y[:, :, :, 5:].isfinite().all()
        table = torch.zeros(2, 2 * Sk + 1, device="cuda")
        pos = Sk - 1 if Sq == 1 else 0
        if Sq == 1:   # a score of -inf hides a key, whatever its value
            table[:, 9 - pos + Sk] = table[:, 11 - pos + Sk] = -math.inf
            assert rt.attention(q, k, v, scale=1.0, dist_bias=table).isfinite().all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_a_nan_that_all_rows_see_costs_little(bad):
    """It took 350 ms where every row was computed again."""
    from edge_maskgit_b200 import runtime as rt
    q, k, v = qkv(1, 4096, 4096, 32, 8, 128, BF16)
    v[0, 100] = bad
    rt.attention(q, k, v, causal=True)
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    e[0].record()
    y = rt.attention(q, k, v, causal=True)
    e[1].record()
    torch.cuda.synchronize()
    assert not y[0, 100:].isfinite().any() and y[0, :100].isfinite().all()
    assert e[0].elapsed_time(e[1]) < 60.0
