"""GPU: cube_sample_rows (csrc/sample.hip) through cube_amd.hip.sample_rows, against the 64-bit oracle.

A token is a decision: it has to equal the oracle's wherever u lies further than 2^-36 of the total from the border between two
candidates (weights are rounded at 2^-41 of the largest or finer for the vocabularies here, the oracle's own running sum at 2^-52
per step; random u lie closer about once in 10^5 rows here, and those rows are not counted).  prob is rounded to fp32 once: 2^-23 of
itself, and 2^-36 of the total for the sums."""
import numpy as np
import pytest
import torch

from cube_amd import hip
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NEAR = 2.0 ** -36


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


def check(z, u, T=1.0, k=0, p=1.0, m=0.0, sure=False):
    """z [M, V] and u [M] on the GPU; settings: numbers or arrays of M.  sure: no row may lie near a border."""
    M = z.shape[0]

    def arg(x, t):
        return torch.tensor(np.asarray(x), dtype=t, device=z.device) if np.ndim(x) else x
    token, prob = hip.sample_rows(z, u, temperature=arg(T, torch.float32), top_k=arg(k, torch.int32), top_p=arg(p, torch.float32),
                                  min_p=arg(m, torch.float32))
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    zz, uu = z.detach().cpu().double().numpy(), u.cpu().numpy()
    f = lambda x, r: float(np.float32(x[r] if np.ndim(x) else x))  # noqa: E731
    near = 0
    for r in range(M):
        kk = int(k[r] if np.ndim(k) else k)
        et, ep, d = oo.sample_row(zz[r], uu[r], f(T, r), kk, f(p, r), f(m, r))
        if d < NEAR and token[r] != et:
            near += 1
            continue
        assert token[r] == et, (r, token[r], et, d)
        assert abs(prob[r] - ep) <= 2.0 ** -23 * ep + NEAR, (r, prob[r], ep)
    assert near <= (0 if sure else 1 + M // 1000), near
    return token


def logits(M, V, t, dev, seed=0, scale=2.5, pad=0, col=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(M, col + V + pad, generator=g) * scale).to(TYPES[t]).to(dev)
    return z[:, col:col + V], torch.rand(M, generator=g, dtype=torch.float64).to(dev)


SIZES = [(5, 1), (9, 2), (40, 63), (40, 64), (40, 65), (70, 102), (20, 255), (20, 256), (20, 257), (20, 511), (20, 513), (8, 1000), (6, 4097), (5, 9000),
         (4, 4096), (3, 32003), (2, 32768), (2, 32769), (2, 100000), (1, 250002), (300, 33000)]
SETTINGS = [dict(), dict(T=0.7), dict(k=1), dict(k=5), dict(k=50), dict(p=0.9), dict(p=0.3, T=1.5), dict(m=0.05), dict(T=0.8, k=40, p=0.95, m=0.02),
            dict(k=1500, p=0.99), dict(T=0.0), dict(p=0.0), dict(m=1.0), dict(T=50.0, p=0.99)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V", SIZES)
def test_sizes_and_types(dev, M, V, t):
    for i, s in enumerate(SETTINGS):
        z, u = logits(M, V, t, dev, seed=100 * i + V)
        check(z, u, **s)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [102, 3000, 40000])
def test_every_row_its_own_settings(dev, V, t):
    M = 60
    rng = np.random.default_rng(V)
    z, u = logits(M, V, t, dev, seed=7)
    T = rng.choice([0.0, 0.5, 0.9, 1.0, 2.0, -1.0, np.nan], M)
    k = rng.choice([0, -3, 1, 2, 17, 60, V - 1, V, V + 5, 2 ** 31 - 1], M)
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 1.0, 2.0, -1.0], M)
    m = rng.choice([0.0, 0.01, 0.2, 1.0, 3.0, -1.0], M)
    check(z, u, T, k, p, m)


@pytest.mark.parametrize("V", [3, 100, 300, 5000, 60000])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_masked_rows(dev, V, t):
    """-inf, NaN and the type's lowest value among the logits; rows of which nothing, one candidate, or only ties are left."""
    ty = TYPES[t]
    z, u = logits(9, V, t, dev, seed=3)
    low = torch.finfo(ty).min
    z[0] = -np.inf
    z[1] = np.nan
    z[2] = -np.inf
    z[2, V - 1] = -5.0
    z[3] = low
    z[4, ::2] = low
    z[5, 1:] = -np.inf
    z[6, ::3] = np.nan
    z[7] = low
    z[7, 1] = 0.0
    z[8, ::2] = -np.inf
    for s in SETTINGS:
        tok = check(z, u, **s)
        assert tok[0] == -1 and tok[1] == -1 and tok[2] == V - 1 and tok[5] == 0 and tok[7] == 1


@pytest.mark.parametrize("V", [5, 100, 400, 7000, 60001])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_infinite_and_huge_logits(dev, V, t):
    """+inf takes all the weight, several share it; finite logits as far apart as the type goes do not overflow."""
    ty = TYPES[t]
    z, _ = logits(4, V, t, dev, seed=4)
    u = torch.tensor([0.1, 0.6, 0.9, 0.5], dtype=torch.float64, device=dev)
    z[0, 2] = np.inf
    z[1, 1] = np.inf
    z[1, 4] = np.inf
    z[2, 3] = torch.finfo(ty).max
    z[2, 0] = torch.finfo(ty).min
    z[3] = torch.finfo(ty).max
    for s in (dict(), dict(p=0.9), dict(k=3), dict(m=0.1), dict(T=1e-30), dict(T=1e-40)):
        tok = check(z, u, sure=True, **s)
        assert tok[0] == 2 and tok[1] in (1, 4) and tok[2] == 3
    tok, prob = hip.sample_rows(z, u, temperature=float("inf"))
    assert tok[0] == 2 and tok[1] == 4 and prob[1] == 0.5


@pytest.mark.parametrize("V", [7, 200, 300, 2000, 30000, 60000])
def test_ties_go_to_the_lowest_index(dev, V):
    """All logits equal (and a mix of -0 and +0): top-k keeps the first k, the running sum is the index."""
    z = torch.zeros(5, V, device=dev)
    z[:, ::2] = -0.0
    u = torch.tensor([0.0, 0.24, 0.5001, 0.75003, 1.0 - 2.0 ** -53], dtype=torch.float64, device=dev)
    k = max(1, V // 3)
    check(z, u)
    tok = check(z, u, k=k)
    assert tok.max() == k - 1 and tok[0] == 0
    check(z, u, p=0.4)
    few = torch.randint(0, 4, (5, V), generator=torch.Generator().manual_seed(V)).float().to(dev)   # four values, many ties each
    for s in (dict(), dict(k=k), dict(k=V // 2 + 1, p=0.9), dict(p=0.37), dict(m=0.3)):
        check(few, u, **s)
        check(few.bfloat16(), u, **s)


@pytest.mark.parametrize("V", [200, 3000, 50000])
def test_values_next_to_each_other(dev, V):
    """f32 logits that differ in the last bits only, and rows that differ from one another beyond bf16's precision."""
    base = torch.full((4, V), 5.0)
    base += torch.randint(0, 8, base.shape, generator=torch.Generator().manual_seed(0)) * 2.0 ** -21
    _, u = logits(4, 10, "f32", dev, seed=1)
    for s in (dict(), dict(k=100), dict(p=0.5), dict(k=700, p=0.6)):
        check(base.to(dev), u, **s)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,col,pad", [(102, 3, 5), (1001, 1, 2), (5000, 7, 1), (20001, 0, 3), (70001, 1, 2)])
def test_strided_and_unaligned_rows(dev, V, col, pad, t):
    z, u = logits(7, V, t, dev, seed=2, col=col, pad=pad)
    for s in (dict(), dict(k=20, p=0.9), dict(p=0.8), dict(m=0.1)):
        a = check(z, u, **s)
        b, _ = hip.sample_rows(z.contiguous(), u, temperature=s.get("T", 1.0), top_k=s.get("k", 0), top_p=s.get("p", 1.0), min_p=s.get("m", 0.0))
        np.testing.assert_array_equal(a, b.cpu().numpy())


def test_random_numbers_at_and_beyond_the_ends(dev):
    z, _ = logits(1, 500, "f32", dev, seed=5)
    z = z.expand(6, 500).contiguous()
    u = torch.tensor([0.0, -1.0, 1.0 - 2.0 ** -53, 1.0, 7.0, float("nan")], dtype=torch.float64, device=dev)
    tok = hip.sample_rows(z, u)[0].cpu().numpy()
    order = oo.candidates(z[0].cpu().double().numpy())
    assert tok[0] == tok[1] == tok[5] == order[0] and tok[2] == tok[3] == tok[4] == order[-1]


@pytest.mark.parametrize("V", [100, 3000])
def test_frequencies(dev, V):
    """Evenly spread u give every candidate its share: counts differ from n * prob by less than 1 (a span of length L holds
    floor or ceil of n * L evenly spread points)."""
    n = 20000
    z, _ = logits(1, V, "f32", dev, seed=6, scale=1.0)
    u = (torch.arange(n, dtype=torch.float64, device=dev) + 0.5) / n
    tok, prob = hip.sample_rows(z.expand(n, V).contiguous(), u, temperature=0.9, top_k=60)
    cnt = np.bincount(tok.cpu().numpy(), minlength=V)
    zz = z[0].cpu().double().numpy()
    keep = oo.candidates(zz)[:60]
    w = np.exp(zz[keep] / float(np.float32(0.9)))
    share = np.zeros(V)
    share[keep] = w / w.sum()
    assert (np.abs(cnt - n * share) < 1 + 1e-6).all()


def test_row_offsets_past_32_bits(dev):
    """Rows whose elements lie beyond 2^32 bytes."""
    V = 1 << 21
    z = torch.zeros(1100, V, dtype=torch.bfloat16, device=dev)
    z[-1, 77], z[0, 5], z[1024, V - 1] = 60.0, 60.0, 60.0
    tok, _ = hip.sample_rows(z[[0, 1024, 1099]], torch.full((3,), 0.5, dtype=torch.float64, device=dev))
    assert tok.tolist() == [5, V - 1, 77]
    tok, _ = hip.sample_rows(z, torch.full((1100,), 0.5, dtype=torch.float64, device=dev), top_k=1)
    assert tok[[0, 1, 1024, 1099]].tolist() == [5, 0, V - 1, 77]


@pytest.mark.parametrize("M,V", [(64, 102), (3, 50000), (200, 20000)])
def test_streams_graphs_and_repeats(dev, M, V):
    """The same tokens every time, on another stream, and from two graphs replayed in turn between eager calls."""
    z, u = logits(M, V, "bf16", dev, seed=8)
    kw = [dict(top_p=0.9), dict(top_k=50, temperature=0.8)]
    first = [hip.sample_rows(z, u, **k) for k in kw]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [hip.sample_rows(z, u, **k) for k in kw]
    side.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for k in kw:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(hip.sample_rows(z, u, **k))
        graphs.append(g)
    for turn in range(3):
        z.copy_(torch.randn(M, V, device=dev) * 2)
        u.copy_(torch.rand(M, dtype=torch.float64, device=dev))
        eager = [hip.sample_rows(z, u, **k) for k in kw]
        for g in (graphs if turn % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        for e, o in zip(eager, outs):
            assert torch.equal(e[0], o[0]) and torch.equal(e[1], o[1])


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_the_longest_row(dev, t):
    """2^22 logits, the most a row may have; one more is refused."""
    V = 1 << 22
    z, u = logits(2, V, t, dev, seed=9)
    for s in (dict(), dict(k=50, p=0.9), dict(p=0.6), dict(m=0.01, T=0.7)):
        check(z, u, **s)
    with pytest.raises(hip.CubeHipError):
        hip.sample_rows(torch.zeros(1, V + 1, dtype=TYPES[t], device=dev), u[:1])


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,k", [(102, 101), (9000, 8999), (32768, 20000), (100000, 30000), (100000, 99999)])
def test_limits_near_the_row(dev, V, k, t):
    """A top-k of thousands, where the kept set is longer than any list the kernels sort."""
    z, u = logits(4, V, t, dev, seed=V + k)
    check(z, u, k=k)
    check(z, u, k=k, p=0.9, T=2.0)


@pytest.mark.parametrize("M,V", [(32, 33000), (33, 33000), (32, 262144), (32, 262145), (60, 33000)])
def test_f16_rows_around_the_change_of_form(dev, M, V):
    """Few f16 rows go another way than many: the same tokens from both, for the same rows."""
    z, u = logits(64, V, "f16", dev, seed=21)
    for s in (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.7), dict(min_p=0.02)):
        many, few = hip.sample_rows(z, u, **s), hip.sample_rows(z[:M], u[:M], **s)
        assert torch.equal(few[0], many[0][:M])
        np.testing.assert_allclose(few[1].cpu(), many[1][:M].cpu(), rtol=2.0 ** -22)
    check(z[:2], u[:2], p=0.8)
    flat = torch.zeros(M, V, dtype=torch.float16, device=dev)       # one value: the list runs over
    check(flat[:2], u[:2], p=0.5)
    assert torch.equal(hip.sample_rows(flat, u[:M], top_p=0.5)[0], hip.sample_rows(flat.repeat(3, 1), u[:M].repeat(3), top_p=0.5)[0][:M])


@pytest.mark.parametrize("M,V", [(70_000_001, 2), (17_000_003, 257)])
def test_more_rows_than_a_launch_has_threads_for(dev, M, V):
    """The arg-max and a draw of two candidates in rows spread over tens of millions, settings and random numbers per row."""
    z = torch.full((M, V), -50.0, dtype=torch.bfloat16, device=dev)
    at = torch.arange(M, device=dev) % V
    z[torch.arange(M, device=dev), at] = 2.0
    u = torch.full((M,), 0.5, dtype=torch.float64, device=dev)
    T = torch.ones(M, device=dev)
    T[::2] = 0.0
    token, prob = hip.sample_rows(z, u, temperature=T)
    assert torch.equal(token.long(), at) and bool((prob == 1).all())


def test_two_streams_at_once(dev):
    """Calls of every form on two streams with nothing between them."""
    cases = [logits(M, V, t, dev, seed=11) + (kw,) for M, V, t in ((500, 102, "f32"), (20, 5000, "bf16"), (8, 60000, "f32"), (8, 60000, "bf16"), (4, 60000, "f16"))
             for kw in (dict(top_p=0.9), dict(top_k=40))]
    want = [hip.sample_rows(z, u, **kw) for z, u, kw in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for turn in range(5):
        for i, (z, u, kw) in enumerate(cases):
            with torch.cuda.stream(streams[(turn + i) % 2]):
                got.append((i, hip.sample_rows(z, u, **kw)))
    for s in streams:
        s.synchronize()
    for i, (token, prob) in got:
        assert torch.equal(token, want[i][0]) and torch.equal(prob, want[i][1])


def test_refusals_on_tensors(dev):
    z, u = logits(4, 50, "f32", dev)
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=1.5), dict(top_k=float("inf")), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0),
                dict(top_k=torch.zeros(4, device=dev)), dict(top_p=torch.zeros(3, device=dev)), dict(min_p=torch.zeros(4)),
                dict(temperature=torch.zeros(8, device=dev)[::2])):
        with pytest.raises(ValueError):
            hip.sample_rows(z, u, **bad)
    for bu in (u.float(), u[:3], u.cpu()):
        with pytest.raises(ValueError):
            hip.sample_rows(z, bu)
    with pytest.raises(ValueError):
        hip.sample_rows(z.t(), u)
    with pytest.raises(ValueError, match="gradient"):
        hip.sample_rows(z.clone().requires_grad_(), u)
    assert hip.sample_rows(z[:0], u[:0])[0].shape == (0,)


def test_a_layer_and_the_sampler_behind_it(dev):
    """Hidden states -> 8-bit output projection -> logits -> tokens, as a decoder uses them: every token is one that the oracle draws
    from the logits that the layer gave, and those are the oracle's within the product's own rounding."""
    from tests.test_gpu_fp8 import close
    g = torch.Generator().manual_seed(12)
    h = torch.randn(24, 300, generator=g).to(dev)
    w = hip.quant_fp8((torch.randn(1500, 300, generator=g) / 4).to(dev))
    bias = torch.randn(1500, generator=g).to(dev)
    u = torch.rand(24, generator=g, dtype=torch.float64).to(dev)
    z = hip.linear_fp8(h, w, bias)
    v, e = oo.quant(h.cpu().double().numpy())
    wv = oo.rows_value(*oo.unpack(w.q.cpu().numpy(), w.scale.cpu().numpy(), 300))
    want, mag = oo.gemm(oo.rows_value(v, e), wv, bias.cpu().double().numpy())
    close(z.cpu().double().numpy(), want, mag, 300, "f32")
    check(z, u, T=0.8, k=40, p=0.95)
    check(z.bfloat16(), u, p=0.9, m=0.05)
