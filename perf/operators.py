"""What the 8-bit floating-point Linear operators and the sampler are measured on: cases, inputs, their plain forms and their
values in 64 bits.  `own` selects the framework's entry points (cube_amd.hip) instead of the plain forms."""
import functools
import math
import os
import sys

import torch

own = False

BLOCK = 128          # columns that share one scale
TOP = 448.0          # largest e4m3 value
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


@functools.lru_cache(maxsize=1)
def _hip():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nlp-cube_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cube_amd import hip
    return hip


# ---- cases ---------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # hidden states of one 33-piece sentence, the LM encoder's width in the K = 13 x 768 configuration
        {"name": "quant sentence", "op": "quant", "M": 33, "K": 768, "type": "f32", "pad": 0},
        # the activations of a large batch before a wide layer
        {"name": "quant large", "op": "quant", "M": 16384, "K": 4096, "type": "bf16", "pad": 0},
        # one fastText layer (300 wide -> 500) over a ragged batch: K is no multiple of the block
        {"name": "gemm ragged", "op": "gemm", "M": 1001, "N": 500, "K": 300, "type": "f32", "act": "tanh"},
        # a square encoder layer over the 8192 words of a full batch
        {"name": "gemm words", "op": "gemm", "M": 8192, "N": 768, "K": 768, "type": "bf16", "act": "none"},
        # the largest: a 4096-wide layer over 8192 rows
        {"name": "gemm large", "op": "gemm", "M": 8192, "N": 4096, "K": 4096, "type": "bf16", "act": "none"},
        # one token through a 4096-wide layer
        {"name": "linear token", "op": "linear", "M": 1, "N": 4096, "K": 4096, "type": "bf16", "act": "none", "pad": 0},
        # one sentence through an encoder layer
        {"name": "linear sentence", "op": "linear", "M": 33, "N": 768, "K": 768, "type": "f32", "act": "none", "pad": 0},
        # the first layer of the external-embedding MLP (768 -> 500) over 8192 words
        {"name": "linear words", "op": "linear", "M": 8192, "N": 500, "K": 768, "type": "f32", "act": "tanh", "pad": 0},
        # a decoding step of the lemmatizer: 8192 words, 102 characters, no filter but the temperature
        {"name": "sample characters", "op": "sample", "M": 8192, "V": 102, "type": "f32", "pad": 6, "kind": "plain"},
        # one request over a sub-word vocabulary, the usual top-k / top-p request
        {"name": "sample token", "op": "sample", "M": 1, "V": 250002, "type": "bf16", "pad": 0, "kind": "topk"},
        # a serving batch of requests with settings of their own (greedy, top-k, top-p, min-p, none)
        {"name": "sample mixed", "op": "sample", "M": 64, "V": 32003, "type": "f32", "pad": 0, "kind": "mixed"},
        # the largest: whole-vocabulary top-p for a full batch
        {"name": "sample large", "op": "sample", "M": 128, "V": 250002, "type": "bf16", "pad": 0, "kind": "topp"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "linear", "sample"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op == "quant":
        K = _log(rng, 40, 8000)
        M = _log(rng, 1, min(16384, 16384 * 4096 // K))
        return {"op": op, "M": M, "K": K, "type": t, "pad": rng.choice([0, 0, 3, 8])}
    if op == "sample":
        V = _log(rng, 20, 250002)
        M = _log(rng, 1, max(1, min(8192, 128 * 250002 // V)))
        return {"op": op, "M": M, "V": V, "type": t, "pad": rng.choice([0, 0, 1, 8]),
                "kind": rng.choice(["plain", "topk", "topp", "minp", "mixed"])}
    N, K = _log(rng, 16, 8000), _log(rng, 40, 8000)
    M = _log(rng, 1, max(1, min(8192, 8192 * 4096 * 4096 // (N * K))))
    act = rng.choice(["none", "tanh", "relu"])
    c = {"op": op, "M": M, "N": N, "K": K, "type": t, "act": act}
    if op == "linear":
        c["M"] = M if rng.random() < 0.5 else min(M, _log(rng, 1, 64))
        c["pad"] = rng.choice([0, 0, 3, 8])
    return c


def work(case):
    M, t = case["M"], SIZE[case["type"]]
    if case["op"] == "sample":
        V = case["V"]
        return {"bytes": M * (V * t + 8 + 16 + 8), "flops": 10 * M * V}
    K = case["K"]
    kb = -(-K // BLOCK)
    if case["op"] == "quant":
        return {"bytes": M * (K * t + kb * BLOCK + kb), "flops": 3 * M * K}
    N = case["N"]
    a = M * K * t if case["op"] == "linear" else M * (K + kb)
    return {"bytes": a + N * (K + kb) + M * N * t + 4 * N, "flops": 2 * M * N * K}


# ---- the number format, in plain torch operations ------------------------------------------------------------------------

def _blocks(x):
    """[M, K] -> [M, KB, 128], zeros behind the last column."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    return torch.nn.functional.pad(x, (0, kb * BLOCK - K)).reshape(M, kb, BLOCK)


def _plain_quant(x):
    """x [M, K] -> (e4m3 [M, KB, 128], exponents int32 [M, KB]).  The exponent is the smallest with max|x| <= 448 * 2^e, the
    product with 2^-e is exact, so the one rounding is the cast's (nearest, ties to even)."""
    b = _blocks(x.float())
    m, e = torch.frexp(b.abs().amax(2))                    # a = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(m == 0, torch.full_like(e, -127), e).clamp(min=-127).to(torch.int32)
    return torch.ldexp(b, -e[:, :, None]).to(torch.float8_e4m3fn), e


def _pack(q, e):
    """The framework's layout of quantised rows: bytes [M, KB*128] and int32 [ceil(KB/4), M], byte j of a word = block 4i+j."""
    M, kb = e.shape
    s = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -kb % 4)).contiguous().view(torch.int32)
    return q.reshape(M, kb * BLOCK).view(torch.uint8), s.t().contiguous()


def _exponents(s, kb):
    """int32 [ceil(KB/4), M] -> exponents [M, KB]."""
    return s.t().contiguous().view(torch.uint8)[:, :kb].to(torch.int32) - 127


def _values(q, e, to):
    M, kb = e.shape
    v = q.view(torch.float8_e4m3fn).reshape(M, kb, BLOCK).to(to)
    return torch.ldexp(v, e[:, :, None]).reshape(M, kb * BLOCK)


ACT = {"none": lambda y: y, "tanh": torch.tanh, "relu": lambda y: torch.clamp(y, min=0)}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _rows(g, M, K, t, pad):
    """Activations with channels of unequal size, as hidden states have them; rows `pad` elements apart from one another."""
    x = torch.randn(M, K + pad, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(K + pad, generator=g, device="cuda"))
    return x.to(TYPES[t])[:, :K]


def _settings(g, M, kind):
    """Per-row temperature, top-k, top-p, min-p of the requests of a batch."""
    r = torch.rand(5, M, generator=g, device="cuda")
    T = 0.6 + 0.8 * r[0]
    k = (1 + 99 * r[1]).to(torch.int32)
    p = 0.8 + 0.18 * r[2]
    m = 0.02 + 0.1 * r[3]
    none = torch.zeros_like(p)
    which = {"plain": 0, "topk": 1, "topp": 2, "minp": 3}.get(kind)
    w = (r[4] * 5).to(torch.int32) if which is None else torch.full((M,), which, dtype=torch.int32, device="cuda")
    T = torch.where(w == 4, none, T)                                    # a greedy request among the others
    k = torch.where(w == 1, k, torch.zeros_like(k))
    p = torch.where((w == 1) | (w == 2), p, none + 1)
    m = torch.where(w == 3, m, none)
    return T, k, p, m


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, t = case["M"], case["type"]
    s = dict(case)
    if case["op"] == "sample":
        V, pad = case["V"], case["pad"]
        z = torch.randn(M, V + pad, generator=g, device="cuda") * 2.5
        hot = torch.randint(0, V, (M, min(V, 8)), generator=g, device="cuda")
        z.scatter_add_(1, hot, 6.0 * torch.rand(hot.shape, generator=g, device="cuda"))   # the words that the context asks for
        z[:, 0] = -math.inf                                                             # a banned token
        s["z"] = z.to(TYPES[t])[:, :V]
        s["u"] = torch.rand(M, generator=g, device="cuda", dtype=torch.float64)
        s["T"], s["k"], s["p"], s["m"] = _settings(g, M, case["kind"])
        return s
    K = case["K"]
    if case["op"] == "quant":
        s["x"] = _rows(g, M, K, t, case["pad"])
        return s
    N = case["N"]
    s["w"] = _pack(*_plain_quant(torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)))   # laid out once, as weights are
    s["bias"] = 0.1 * torch.randn(N, generator=g, device="cuda")
    x = _rows(g, M, K, t, case.get("pad", 0))
    if case["op"] == "linear":
        s["x"] = x
    else:
        s["a"] = _pack(*_plain_quant(x))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------

def _plain_sample(z, u, T, k, p, m):
    z = torch.nan_to_num(z.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    v, order = torch.sort(z, dim=1, descending=True, stable=True)
    V = z.shape[1]
    rank = torch.arange(V, device=z.device)
    greedy = ~(T > 0)
    T = torch.where(greedy, torch.ones_like(T), T).double()[:, None]
    w = torch.exp((v - v[:, :1]) / T)
    w = torch.where(v == v[:, :1], torch.ones_like(w), w)
    w = torch.where(v == -math.inf, torch.zeros_like(w), w)
    k = torch.where((k <= 0) | (k > V), torch.full_like(k, V), k)[:, None]
    w1 = w * (rank < k)
    c = torch.cumsum(w1, 1)
    p = p.double()[:, None]
    keep = (rank < k) & ((p >= 1) | (c - w1 < p * c[:, -1:])) & (w >= m.double().clamp(max=1)[:, None])
    w = w * (keep | (rank == 0))
    c = torch.cumsum(w, 1)
    at = (c <= u[:, None] * c[:, -1:]).sum(1).clamp(max=V - 1)
    at = torch.where(greedy, torch.zeros_like(at), at)[:, None]
    prob = torch.where(greedy[:, None], (w[:, :1] > 0).double(), w.gather(1, at) / c[:, -1:].clamp(min=1e-300))
    token = torch.where(v[:, :1] == -math.inf, torch.full_like(at, -1), order.gather(1, at))
    return {"token": token[:, 0].to(torch.int32), "prob": prob[:, 0].float()}


def _own_run(s):
    hip = _hip()
    op = s["op"]
    if op == "quant":
        a = hip.quant_fp8(s["x"])
        return {"q": a.q.view(torch.float8_e4m3fn), "scale": a.scale}
    if op == "sample":
        token, prob = hip.sample_rows(s["z"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        return {"token": token, "prob": prob}
    w = hip.Fp8Rows(*s["w"], s["K"])
    if op == "linear":
        return {"out": hip.linear_fp8(s["x"], w, s["bias"], act=s["act"])}
    return {"out": hip.gemm_fp8(hip.Fp8Rows(*s["a"], s["K"]), w, s["bias"], act=s["act"], out_dtype=TYPES[s["type"]])}


def run(s):
    if own:
        return _own_run(s)
    op = s["op"]
    if op == "quant":
        q, scale = _pack(*_plain_quant(s["x"]))
        return {"q": q.view(torch.float8_e4m3fn), "scale": scale}
    if op == "sample":
        return _plain_sample(s["z"], s["u"], s["T"], s["k"], s["p"], s["m"])
    kb = -(-s["K"] // BLOCK)
    if op == "linear":
        a = _values(*_plain_quant(s["x"]), torch.float32)
    else:
        a = _values(s["a"][0], _exponents(s["a"][1], kb), torch.float32)
    w = _values(s["w"][0], _exponents(s["w"][1], kb), torch.float32)
    return {"out": ACT[s["act"]](a @ w.t() + s["bias"]).to(TYPES[s["type"]])}


# ---- the same values in 64 bits, from the definitions --------------------------------------------------------------------

def _exact_exponent(a):
    """Smallest e >= -127 with a <= 448 * 2^e: from the logarithm, put right by one where the comparison says so."""
    e = torch.ceil(torch.log2(torch.clamp(a, min=2.0 ** -140) / TOP))
    e = torch.where(a > TOP * torch.exp2(e), e + 1, e)
    e = torch.where(a <= TOP * torch.exp2(e - 1), e - 1, e)
    return e.clamp(min=-127)


def _exact_quant(x):
    b = _blocks(x.double())
    e = _exact_exponent(b.abs().max(2).values)
    y = b / torch.exp2(e)[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6))) - 3)   # 3 bits behind the point, from 2^-6 on
    return torch.round(y / step) * step, e                                                # round: ties to even


def _exact_values(packed, K):
    """The numbers that packed rows stand for, from the bits: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    q, s = packed
    kb = -(-K // BLOCK)
    i = q.to(torch.int64)
    exp, frac = (i >> 3) & 15, (i & 7).double()
    v = torch.where(exp == 0, frac * 2.0 ** -9, (1 + frac / 8) * torch.exp2((exp - 7).double())) * (1 - 2 * (i >> 7)).double()
    e = torch.stack([(s[b // 4].to(torch.int64) >> (8 * (b % 4))) & 255 for b in range(kb)], 1).double() - 127
    return v * torch.exp2(e).repeat_interleave(BLOCK, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        q, e = _exact_quant(s["x"])
        return {"q": q.reshape(q.shape[0], -1), "scale": None}
    if op == "sample":
        z, u = s["z"].double(), s["u"]
        M, V = z.shape
        probs = []
        for r in range(M):          # row by row: sorted candidates, three prefixes, the running sum
            T, k, p, m = (float(s[n][r]) for n in ("T", "k", "p", "m"))
            zs = torch.sort(z[r][z[r] > -math.inf], descending=True, stable=True).values
            if T <= 0:
                probs.append(torch.ones((), device=z.device, dtype=torch.float64))
                continue
            w = torch.exp((zs - zs[0]) / T)
            if 0 < k < len(w):
                w = w[:int(k)]
            if p < 1:
                c = torch.cumsum(w, 0)
                w = w[:int(torch.searchsorted(c, p * c[-1])) + 1]
            w = w[:max(1, int((w >= m).sum()))]
            c = torch.cumsum(w, 0)
            probs.append(w[min(int(torch.searchsorted(c, u[r] * c[-1], right=True)), len(w) - 1)] / c[-1])
        return {"token": None, "prob": torch.stack(probs)}
    K = case["K"]
    if op == "linear":
        q, e = _exact_quant(s["x"])
        a = (q * torch.exp2(e)[:, :, None]).reshape(q.shape[0], -1)
    else:
        a = _exact_values(s["a"], K)
    y = torch.matmul(a, _exact_values(s["w"], K).t()) + s["bias"].double()
    return {"out": torch.tanh(y) if case["act"] == "tanh" else torch.where(y > 0, y, torch.zeros_like(y)) if case["act"] == "relu" else y}
