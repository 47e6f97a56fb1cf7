"""Measured cases of the 16-bit serving operators: attention with shaped scores, the linear
layer with its epilogue, and the adjustment of logits before a draw.

Each case runs in two forms on the same inputs: a plain one in elementary float32 torch
operations, and the framework's entry points in ``edge_maskgit_b200.runtime``.

attention   s = scale q.k;  s = cap tanh(s / cap) where cap > 0;  s -= slope |p - j|;
            s += table[clamp(j - p, -R, R) + R];  key j of a row at position p is seen where
            j < k_len, the document numbers are equal and not negative, and (causal) j <= p or
            j < prefix;  out = softmax(s) v, and zeros for a row that sees nothing.
linear      y = act(x W^T + bias) + resid.
logits      z = z > 0 ? z / rep : z rep for a token that the row's history holds (c times),
            z -= freq c + pres [c > 0];  z += bias;  -inf where the row's allowed bit is 0.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------ cases
def _attn(**kw):
    case = dict(op="attention", dtype="bf16", B=1, Sq=1, Sk=1, Hq=1, Hkv=1, D=64, cap=0.0, slopes=False, reach=0,
                causal=False, prefix=0, docs=0, ragged=False, packed=False)
    case.update(kw)
    return case


def _linear(**kw):
    case = dict(op="linear", dtype="bf16", M=1, K=64, N=64, bias=True, act=0, resid=False)
    case.update(kw)
    return case


def _logits(**kw):
    case = dict(op="logits", dtype="f32", R=1, V=32, L=1, bias="none", allowed="none")
    case.update(kw)
    return case


def listed():
    return [
        # one 256 x 256 image of the transformer (class token and 16 x 16 codes): a call where latency counts
        _attn(name="attn_image", dtype="f16", Sq=257, Sk=257, Hq=16, Hkv=16, D=48, reach=32, packed=True),
        # images of several sizes packed into one long row, each attending to itself only
        _attn(name="attn_documents", Sq=4097, Sk=4097, Hq=16, Hkv=16, D=48, reach=128, docs=13, packed=True),
        # a padded batch with a decaying bias by distance
        _attn(name="attn_slopes", dtype="f16", B=4, Sq=2001, Sk=2001, Hq=16, Hkv=16, D=64, slopes=True, causal=True,
              ragged=True),
        # a long prompt with a two-way prefix, shared key heads and capped scores
        _attn(name="attn_prefix", Sq=8192, Sk=8192, Hq=32, Hkv=8, D=128, cap=50.0, causal=True, prefix=1000),
        # one new token against one sequence's cache: latency
        _attn(name="attn_step", Sk=4096, Hq=32, Hkv=8, D=128, causal=True),
        # one new token for each of a batch of sequences of unequal length: bytes of the cache
        _attn(name="attn_step_batch", B=32, Sk=16385, Hq=32, Hkv=8, D=128, cap=30.0, causal=True, ragged=True),
        # one token through a square layer: the weight's bytes
        _linear(name="linear_step", M=1, K=4096, N=4096, act=2),
        # the q | k | v projection of one image
        _linear(name="linear_image", dtype="f16", M=257, K=768, N=2304),
        # the logits of one long sequence: an odd number of columns
        _linear(name="linear_head", dtype="f16", M=4097, K=768, N=2025),
        # the wide layer of a long batch: the largest product
        _linear(name="linear_wide", M=8192, K=4096, N=14336, act=1, resid=True),
        # every position of one image before its draw
        _logits(name="logits_image", R=257, V=2025, L=257, bias="shared", allowed="shared"),
        # a large batch over a large vocabulary, each row with its own grammar
        _logits(name="logits_batch", dtype="bf16", R=256, V=128257, L=4096, bias="shared", allowed="rows"),
    ]


def _spread(rng, lo, hi):
    """An integer from lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "step", "linear", "linear", "logits"])
    if kind == "linear":
        M, K, N = _spread(rng, 1, 8192), 8 * _spread(rng, 8, 1024), _spread(rng, 16, 16384)
        while M * K * N > 8192 * 4096 * 14336:
            M = max(1, M // 2)
        return _linear(dtype=rng.choice(["f16", "bf16"]), M=M, K=K, N=N, bias=rng.random() < 0.7, act=rng.randrange(3),
                       resid=rng.random() < 0.5)
    if kind == "logits":
        R, V = _spread(rng, 1, 512), _spread(rng, 1000, 150000)
        while R * V > 256 * 128257:
            R = max(1, R // 2)
        return _logits(dtype=rng.choice(["f32", "f16", "bf16"]), R=R, V=V, L=_spread(rng, 1, 4096),
                       bias=rng.choice(["none", "shared", "rows"]), allowed=rng.choice(["none", "shared", "rows"]))
    Hkv, group = rng.choice([(16, 1), (8, 4), (4, 8), (2, 7), (1, 16), (12, 1)])
    case = _attn(dtype=rng.choice(["f16", "bf16"]), Hq=Hkv * group, Hkv=Hkv, D=rng.choice([32, 48, 64, 80, 96, 128]),
                 cap=rng.choice([0.0, 0.0, 20.0, 50.0]), causal=rng.random() < 0.6)
    if kind == "step":
        case.update(B=_spread(rng, 1, 32), Sq=rng.choice([1, 1, 1, 2, 5]), Sk=_spread(rng, 64, 32768), ragged=rng.random() < 0.6)
        while case["B"] * case["Sk"] * case["Hkv"] * case["D"] > 32 * 16385 * 8 * 128:
            case["B"] = max(1, case["B"] // 2)
    else:
        S = _spread(rng, 17, 8192)
        case.update(Sq=S, Sk=S, packed=case["Hq"] == case["Hkv"] and rng.random() < 0.5)
        case["B"] = _spread(rng, 1, max(1, min(8, 32 * 8192 * 8192 // (case["Hq"] * S * S))))
        if rng.random() < 0.35:
            case["docs"] = rng.randint(1, max(1, min(40, S // 8)))
        elif rng.random() < 0.4:
            case["ragged"] = True
        if case["causal"] and rng.random() < 0.5:
            case["prefix"] = rng.randint(1, S)
    bias = rng.choice(["none", "slopes", "table"])
    case["slopes"] = bias == "slopes"
    case["reach"] = rng.choice([16, 128, 1000]) if bias == "table" else 0
    return case


def _lengths(case):
    """Keys that each batch row holds."""
    if not case["ragged"]:
        return [case["Sk"]] * case["B"]
    rng = random.Random(case["Sk"] * 131 + case["B"])
    return [max(case["Sq"], int(case["Sk"] * rng.uniform(0.5, 1.0))) for _ in range(case["B"])]


def _documents(case):
    """Lengths of the documents that share a row, and of the padding behind them."""
    rng = random.Random(case["Sk"] * 17 + case["docs"])
    shares = [rng.uniform(0.3, 1.7) for _ in range(case["docs"])]
    used = case["Sk"] - case["Sk"] // 50
    lens = [max(1, int(used * s / sum(shares))) for s in shares]
    return lens, case["Sk"] - sum(lens)


# ----------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0):
        return (torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=gen)).mul_(std)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return dict(case=case, x=normal(M, K), w=normal(N, K, std=K ** -0.5),
                    bias=normal(N, dtype=torch.float32, std=0.1) if case["bias"] else None,
                    resid=normal(M, N) if case["resid"] else None)
    if case["op"] == "logits":
        R, V, L = case["R"], case["V"], case["L"]
        words = (V + 31) // 32
        state = dict(case=case, logits=normal(R, V, std=3.0), bias=None, allowed=None)
        # a history repeats itself: tokens are drawn from a small part of the vocabulary; lengths differ by row
        state["history"] = ints(0, max(2, V // 16), R, L)
        state["hist_len"] = ints(0, L + 1, R)
        state["penalties"] = torch.stack([1.0 + 0.5 * torch.rand(R, generator=gen, device="cuda"),
                                          0.5 * torch.rand(R, generator=gen, device="cuda"),
                                          0.5 * torch.rand(R, generator=gen, device="cuda")], 1).contiguous()
        if case["bias"] != "none":
            state["bias"] = normal(*((V,) if case["bias"] == "shared" else (R, V)), dtype=torch.float32)
        if case["allowed"] != "none":
            rows = () if case["allowed"] == "shared" else (R,)
            state["allowed"] = ints(-2 ** 31, 2 ** 31 - 1, *rows, words) | ints(-2 ** 31, 2 ** 31 - 1, *rows, words)
        return state
    B, Sq, Sk, Hq, Hkv, D = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    if case["packed"]:   # q | k | v side by side, as a projection leaves them
        q, k, v = normal(B, Sq, 3, Hq, D).unbind(2)
    else:
        q, k, v = normal(B, Sq, Hq, D), normal(B, Sk, Hkv, D), normal(B, Sk, Hkv, D)
    state = dict(case=case, q=q, k=k, v=v, scale=D ** -0.5, slopes=None, table=None, prefix=None, k_len=None, q_pos=None,
                 doc=None)
    if case["slopes"]:
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device="cuda", dtype=torch.float32) / Hq)
    if case["reach"]:
        state["table"] = normal(Hq, 2 * case["reach"] + 1, dtype=torch.float32)
    if case["prefix"]:
        state["prefix"] = torch.full((B,), case["prefix"], device="cuda", dtype=torch.int32)
    if case["ragged"]:
        state["k_len"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        if Sq < Sk:   # the new tokens are the last of their sequence
            state["q_pos"] = state["k_len"] - Sq
    if case["docs"]:
        lens, rest = _documents(case)
        ids = [i for i, n in enumerate(lens) for _ in range(n)] + [-1] * rest
        state["doc"] = torch.tensor(ids, device="cuda", dtype=torch.int32).expand(B, Sk).contiguous()
    return state


# ------------------------------------------------------------------------------------- runs
def run(s):
    case = s["case"]
    if own:
        from edge_maskgit_b200 import runtime as rt
        if case["op"] == "linear":
            return rt.linear(s["x"], s["w"], bias=s["bias"], act=case["act"], resid=s["resid"])
        if case["op"] == "logits":
            return rt.logits_adjust(s["logits"], history=s["history"], hist_len=s["hist_len"], penalties=s["penalties"],
                                    bias=s["bias"], allowed=s["allowed"])
        return rt.attention(s["q"], s["k"], s["v"], scale=s["scale"], cap=case["cap"], slopes=s["slopes"],
                            dist_bias=s["table"], causal=case["causal"], prefix=s["prefix"], k_len=s["k_len"],
                            q_pos=s["q_pos"], doc_q=s["doc"], doc_k=s["doc"])
    if case["op"] == "linear":
        return _plain_linear(s)
    if case["op"] == "logits":
        return _plain_logits(s)
    return _plain_attention(s)


def _plain_linear(s):
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    if act == 1:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif act == 2:
        y = y / (1.0 + torch.exp(-y))
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(s["x"].dtype)


def _plain_logits(s):
    case = s["case"]
    z = s["logits"].float()
    R, V = z.shape
    held = torch.arange(case["L"], device=z.device)[None] < s["hist_len"][:, None]
    count = torch.zeros(R, V + 1, device=z.device)
    count.scatter_add_(1, torch.where(held, s["history"].long(), V), torch.ones_like(held, dtype=torch.float32))
    count = count[:, :V]
    rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
    seen = count > 0
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - (freq * count + pres * seen)
    if s["bias"] is not None:
        z = z + s["bias"]
    if s["allowed"] is not None:
        at = torch.arange(V, device=z.device)
        bit = (s["allowed"][..., at // 32] >> (at % 32)) & 1
        z = torch.where(bit == 1, z, -math.inf)
    return z.to(s["logits"].dtype)


def _seen(s, case, dev):
    """[B or 1][Sq][Sk] truth values, or None where every row sees every key; and j - p."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    first = s["q_pos"] if s["q_pos"] is not None else torch.full((1,), Sk - Sq, device=dev)
    p = first[:, None] + torch.arange(Sq, device=dev)
    j = torch.arange(Sk, device=dev)
    dist = j[None, None, :] - p[:, :, None]
    ok = None
    if case["causal"]:
        ok = dist <= 0
        if s["prefix"] is not None:
            ok = ok | (j[None, None, :] < s["prefix"][:, None, None])
    if s["k_len"] is not None:
        m = j[None, None, :] < s["k_len"][:, None, None]
        ok = m if ok is None else ok & m
    if s["doc"] is not None:
        m = (s["doc"][:, :, None] == s["doc"][:, None, :]) & (s["doc"][:, :, None] >= 0)
        ok = m if ok is None else ok & m
    return ok, dist


def _plain_attention(s):
    case = s["case"]
    B, Sq, Sk, Hq, Hkv, D = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    g = Hq // Hkv
    q = s["q"].float().reshape(B, Sq, Hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * Sq, D)
    k = s["k"].float().permute(0, 2, 3, 1)
    v = s["v"].float().permute(0, 2, 1, 3)
    sc = (q @ k).reshape(B, Hq, Sq, Sk) * s["scale"]
    if case["cap"]:
        sc = case["cap"] * torch.tanh(sc / case["cap"])
    ok, dist = _seen(s, case, q.device)
    if s["slopes"] is not None:
        sc = sc - s["slopes"][None, :, None, None] * dist.abs()[:, None].float()
    if s["table"] is not None:
        R = case["reach"]
        sc = sc + s["table"][:, dist.clamp(-R, R) + R].transpose(0, 1)
    if ok is not None:
        sc = torch.where(ok[:, None], sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(B, Hkv, g * Sq, Sk) @ v).reshape(B, Hq, Sq, D)
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 2, 1, 3).to(s["q"].dtype).contiguous()


# ------------------------------------------------------------------------------------- work
def _pairs(case):
    """Seen (row, key) pairs of one head."""
    Sq, Sk = case["Sq"], case["Sk"]

    def block(rows, first, keys):   # rows at positions first.. of `keys` keys
        if not case["causal"]:
            return rows * keys
        lo = min(keys, case["prefix"])
        return sum(min(keys, max(lo, first + i + 1)) for i in range(rows))

    if case["docs"]:
        total, start = 0, 0
        for n in _documents(case)[0]:
            if case["causal"]:
                pre = max(0, min(n, case["prefix"] - start))
                total += sum(max(pre, i + 1) for i in range(n))
            else:
                total += n * n
            start += n
        return case["B"] * total
    return sum(block(Sq, (n if Sq < Sk else Sk) - Sq, n) for n in _lengths(case))


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": size * (M * K + N * K + M * N * (2 if case["resid"] else 1)) + (4 * N if case["bias"] else 0),
                "flops": 2 * M * K * N}
    if case["op"] == "logits":
        R, V, L = case["R"], case["V"], case["L"]
        words = 4 * ((V + 31) // 32)
        more = {"none": 0, "shared": 1, "rows": R}
        return {"bytes": 2 * size * R * V + 4 * R * (L // 2) + more[case["bias"]] * 4 * V + more[case["allowed"]] * words,
                "flops": 6 * R * V}
    B, Sq, Hq, Hkv, D = (case[n] for n in ("B", "Sq", "Hq", "Hkv", "D"))
    keys = B * (case["Sk"] - _documents(case)[1]) if case["docs"] else sum(_lengths(case))
    return {"bytes": size * D * (2 * B * Sq * Hq + 2 * Hkv * keys), "flops": 4 * D * Hq * _pairs(case)}


# ------------------------------------------------------------------------- the 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["act"] == 1:
            y = y * torch.special.ndtr(y)
        elif case["act"] == 2:
            y = y * torch.sigmoid(y)
        return y if s["resid"] is None else y + s["resid"].double()
    if case["op"] == "logits":
        z = s["logits"].double()
        V = case["V"]
        for r in range(case["R"]):
            n = int(s["hist_len"][r])
            c = torch.bincount(s["history"][r, :n].long(), minlength=V).double()
            rep, freq, pres = s["penalties"][r].double().tolist()
            row = z[r]
            row = torch.where(c == 0, row, torch.where(row > 0, row / rep, row * rep)) - c * freq
            row[c > 0] -= pres
            z[r] = row
        if s["bias"] is not None:
            z += s["bias"].double()
        if s["allowed"] is not None:
            shifts = torch.arange(32, device=z.device, dtype=torch.int32)
            bits = ((s["allowed"][..., None] >> shifts) & 1).flatten(-2)[..., :V]
            z.masked_fill_((bits == 0).expand_as(z), -math.inf)
        return z
    Sq, Sk, g = case["Sq"], case["Sk"], case["Hq"] // case["Hkv"]
    out = torch.zeros(case["B"], Sq, case["Hq"], case["D"], dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        n = Sk if s["k_len"] is None else int(s["k_len"][b])
        first = Sk - Sq if s["q_pos"] is None else int(s["q_pos"][b])
        rows = torch.arange(first, first + Sq, device="cuda")[:, None]
        keys = torch.arange(n, device="cuda")[None]
        hide = torch.zeros(Sq, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hide |= (keys > rows) & (keys >= case["prefix"])
        if s["doc"] is not None:
            dq, dk = s["doc"][b, :Sq, None], s["doc"][b, None, :n]
            hide |= (dq != dk) | (dk < 0)
        for h in range(case["Hq"]):
            sc = torch.einsum("id,jd->ij", s["q"][b, :, h].double(), s["k"][b, :n, h // g].double()) * s["scale"]
            if case["cap"]:
                sc = torch.tanh(sc / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                sc -= s["slopes"][h].double() * (rows - keys).abs()
            if s["table"] is not None:
                R = case["reach"]
                sc += s["table"][h].double()[(keys - rows).clamp(-R, R) + R]
            sc.masked_fill_(hide, -math.inf)
            out[b, :, h] = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0) @ s["v"][b, :n, h // g].double()
    return out
