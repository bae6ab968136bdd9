"""GPU: the 8-bit Linear operators, calls that tests/test_gpu_fp8.py does not make.  Its docstring derives the products' tolerances."""
import numpy as np
import pytest
import torch

from cube_amd import hip
from oracle import ops_oracle as oo
from tests.test_gpu_fp8 import TYPES, close, integer_rows, np_, random_rows, rows_from, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


# ---- tanh -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [7, 40, 300])
def test_tanh_of_small_and_large_values(dev, M, t):
    """Every product picks one activation value, so the sums are exact: the magnitudes of e4m3 from 2^-60 to 2^9, both signs.  The kernel's
    tanh is within 1.7 * 2^-23 < 2^-22 of itself; the output type adds half a step of the value (below its normal numbers half the
    smallest subnormal)."""
    mags = oo.e4m3_values()[1:127]
    info = torch.finfo(TYPES[t])
    w = np.zeros((16, 128))
    w[np.arange(16), 8 * np.arange(16)] = np.where(np.arange(16) % 2, -1.0, 1.0)
    w = rows_from(w, np.full((16, 1), 127), 128, dev)
    for byte in list(range(67, 130, 3)) + [118, 119, 120, 121]:
        v = np.zeros((M, 128))
        v[:, ::8] = np.resize(mags, (M, 16))
        got = np_(hip.gemm_fp8(rows_from(v, np.full((M, 1), byte), 128, dev), w, act="tanh", out_dtype=TYPES[t]))
        x = v[:, ::8] * 2.0 ** (byte - 127) * np.where(np.arange(16) % 2, -1.0, 1.0)
        want = np.tanh(x)
        err = 2.0 ** -22 * np.abs(want)
        tol = err + info.eps / 2 * (np.abs(want) + err) + info.smallest_normal * info.eps / 2
        bad = np.abs(got - want) > tol
        assert not bad.any(), (byte, x[bad][:4], got[bad][:4], want[bad][:4])
        assert (np.sign(got[want * 1.0 >= info.smallest_normal * info.eps]) == 1).all()


def test_tanh_at_its_ends(dev):
    """Sums of 0, infinities and NaN through tanh: 0, 1, -1, NaN; and a bias alone, next to where the two formulas meet."""
    w = hip.quant_fp8(torch.ones(6, 128, device=dev))
    x = torch.zeros(40, 128, device=dev)
    edge = np.float32(0.875)
    bias = torch.tensor([0.0, 1e30, -1e30, float(edge), float(np.nextafter(edge, np.float32(0))), -3e-39], device=dev)
    for rows in (x[:3], x):
        got = hip.linear_fp8(rows, w, bias, act="tanh")
        want = np.tanh(np_(bias))
        assert bool((got == got[0]).all())
        np.testing.assert_allclose(np_(got[0]), want, rtol=2.0 ** -22, atol=2.0 ** -149)
    x[1, 5] = float("nan")
    assert bool(torch.isnan(hip.linear_fp8(x, w, bias, act="tanh")[1]).all())


# ---- memory beside memory ---------------------------------------------------------------------------------------------------

def test_arrays_beside_one_another_are_taken(dev):
    """Random layouts of cube_quant_fp8 within one buffer that share no byte: the call is taken and writes what it does elsewhere, and
    nothing else.  (Rows of two distances within one another's range are refused whether or not they meet.)"""
    import random
    rng = random.Random(2)
    size = 1 << 16
    buf = torch.zeros(size, dtype=torch.uint8, device=dev)
    lib, base, taken = hip.load(), buf.data_ptr(), 0
    for _ in range(400):
        M, K = rng.randint(1, 6), rng.randint(1, 140)
        kb = -(-K // 128)
        pitch = 16 * rng.randint(64, 90)                         # x and q as windows of one matrix, or lying one behind the other
        ld_x, ld_q, ld_s = (pitch // 4, pitch, M) if rng.random() < 0.6 else (K + rng.choice([0, 5]), kb * 128 + 16 * rng.choice([0, 9]), M + rng.choice([0, 3]))
        x, q, s = 4 * rng.randint(0, 2000), 16 * rng.randint(0, 600), 4 * rng.randint(0, 3000)
        bx = {x + 4 * ld_x * r + i for r in range(M) for i in range(4 * K)}
        bq = {q + ld_q * r + i for r in range(M) for i in range(kb * 128)}
        bs = {s + i for i in range(4 * M)}
        within = x < q + ld_q * (M - 1) + kb * 128 and q < x + 4 * (ld_x * (M - 1) + K)
        two = M > 1 and 4 * ld_x != ld_q and 4 * K != 4 * ld_x and kb * 128 != ld_q and within
        if bx & bq or bx & bs or bq & bs or two:
            continue
        taken += 1
        v = torch.randn(M, K)
        host = np.full(size, 0xA5, dtype=np.uint8)
        for r in range(M):
            host[x + 4 * ld_x * r: x + 4 * (ld_x * r + K)] = v[r].numpy().view(np.uint8)
        buf.copy_(torch.from_numpy(host))
        assert lib.cube_quant_fp8(base + x, 0, ld_x, M, K, base + q, ld_q, base + s, ld_s, hip.stream_handle()) == 0, lib.cube_last_error()
        want = hip.quant_fp8(v.to(dev))
        for r in range(M):
            host[q + ld_q * r: q + ld_q * r + kb * 128] = want.q[r].cpu().numpy()
        host[s: s + 4 * M] = want.scale[0].cpu().numpy().view(np.uint8)
        np.testing.assert_array_equal(buf.cpu().numpy(), host)
    assert taken > 60


def test_an_output_between_its_inputs(dev):
    """out, bias and weights in one allocation without a gap, and a token vector behind its logits: taken."""
    M, N, K = 70, 64, 256
    buf = torch.zeros(1 << 18, dtype=torch.uint8, device=dev)
    w = hip.quant_fp8(torch.randn(N, K, device=dev))
    q = buf[:N * K].view(N, K)
    s = buf[N * K:N * K + 4 * N].view(torch.int32).view(1, N)
    out = buf[N * K + 4 * N:N * K + 4 * N + 2 * M * N].view(torch.bfloat16).view(M, N)
    bias = buf[N * K + 4 * N + 2 * M * N:][:4 * N].view(torch.float32)
    q.copy_(w.q), s.copy_(w.scale), bias.copy_(torch.randn(N, device=dev))
    x = torch.randn(M, K, device=dev).bfloat16()
    want = hip.linear_fp8(x, w, bias.clone())
    assert torch.equal(hip.linear_fp8(x, hip.Fp8Rows(q, s, K), bias, out=out), want)
    with pytest.raises(hip.CubeHipError, match="overlaps bias"):
        hip.linear_fp8(x, hip.Fp8Rows(q, s, K), buf[N * K + 4 * N:][:4 * N].view(torch.float32), out=out)


# ---- every tile and both of its loops, with 16-bit outputs --------------------------------------------------------------------

def scaled_integers(rng, rows, K, dev):
    """Codes of magnitude up to 3 at scales 1, 2, 4, another for every block of every row: sums of up to 2^15 products (at most 9 * 16
    each) are integers below 2^23, exact in fp32 whatever their order, and lose nothing in the 8-bit instructions (one block, one scale)."""
    kb = -(-K // 128)
    v = rng.integers(-3, 4, (rows, kb * 128)).astype(np.float64)
    v[:, K:] = 0
    return rows_from(v, rng.integers(127, 130, (rows, kb)), K, dev)


# 256x256 tiles by blocks of K (one, more than its two stages, over a change of the scale word, around two); 128x128; 128x64; 64x64 with
# four stages and with wave groups along K
TILES = [(4000, 4050, K) for K in (100, 300, 512, 600, 768, 1100)] + [(5000, 3900, 260), (8192, 768, 768), (8000, 520, 1000), (8192, 768, 100), (2100, 1100, 700),
                                                                      (2100, 1100, 130), (512, 768, 768), (65, 1000, 2500), (300, 260, 1500)]


@pytest.mark.parametrize("M,N,K", TILES)
def test_every_tile_in_16_bits(dev, M, N, K):
    rng = np.random.default_rng(M + N + K)
    a, w = scaled_integers(rng, M, K, dev), scaled_integers(rng, N, K, dev)
    bias = rng.integers(-50, 50, N).astype(np.float32)
    y = (a.float().double() @ w.float().double().t()).cpu() + torch.from_numpy(bias).double()
    for t in (torch.bfloat16, torch.float16, torch.float32):
        got = hip.gemm_fp8(a, w, torch.from_numpy(bias).to(dev), out_dtype=t)
        assert torch.equal(got.cpu(), y.float().to(t)), t


@pytest.mark.parametrize("M,N,K", [(4000, 4050, 600), (8192, 768, 300), (2100, 1100, 300)])
def test_large_tiles_into_strided_rows(dev, M, N, K):
    rng = np.random.default_rng(7)
    a, w = scaled_integers(rng, M, K, dev), scaled_integers(rng, N, K, dev)
    for t in (torch.bfloat16, torch.float16):
        want = hip.gemm_fp8(a, w, out_dtype=t)
        for col, pad in ((1, 2), (8, 8), (0, 1)):
            base = torch.full((M + 2, col + N + pad), -7.0, dtype=t, device=dev)
            hip.gemm_fp8(a, w, out=base[1:M + 1, col:col + N])
            assert torch.equal(base[1:M + 1, col:col + N], want)
            base[1:M + 1, col:col + N] = -7.0
            assert bool((base == -7.0).all())


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 16, 20, 33, 48, 60, 130])
def test_a_vocabulary_in_16_bits(dev, M, t):
    """As the fp32 test of a vocabulary: few rows (a tile of columns a wave) and many."""
    rng = np.random.default_rng(M)
    N, K = 131072 + 77, 260
    w = integer_rows(rng, 1000, K, dev)
    few = w.float().double()
    w = hip.Fp8Rows(w.q.repeat(132, 1)[:N].contiguous(), w.scale.repeat(1, 132)[:, :N].contiguous(), K)
    x = torch.randint(-3, 4, (M, K), generator=torch.Generator().manual_seed(M)).float()
    x[:, ::128] = 448.0                                      # the scale of every block is 1: the small integers stay what they are
    # 448 times at most 3 beside products of at most 9: fewer than 13 bits, nothing is lost
    want = (x.to(dev).double() @ few.t()).repeat(1, 132)[:, :N].float().to(TYPES[t])
    for got in (hip.linear_fp8(x.to(dev).to(TYPES[t]), w), hip.gemm_fp8(hip.quant_fp8(x.to(dev)), w, out_dtype=TYPES[t])):
        assert torch.equal(got, want)


# ---- streams ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("M", [1, 33, 200, 3000])
def test_quantiser_and_product_on_a_side_stream(dev, M, t):
    """The two calls one behind the other on another stream than the tensors were made on: the same bits as on their own, in new memory
    each time; and as one call, where that runs the same product."""
    x = torch.randn(M, 1000, device=dev).to(TYPES[t])
    w = hip.quant_fp8(torch.randn(300, 1000, device=dev))
    first = hip.gemm_fp8(hip.quant_fp8(x), w, out_dtype=TYPES[t])
    v, e = oo.quant(np_(x))
    want, mag = oo.gemm(oo.rows_value(v, e), values(w))
    close(np_(first), want, mag, 1000, t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            got = hip.gemm_fp8(hip.quant_fp8(x), w, out_dtype=TYPES[t])
        side.synchronize()
        assert torch.equal(got, first)
    if M >= 200:
        assert torch.equal(hip.linear_fp8(x, w), first)


@pytest.mark.parametrize("M,N,K,t", [(1001, 500, 300, "f32"), (8192, 768, 768, "bf16"), (4000, 4050, 1100, "bf16"), (1, 4096, 4096, "bf16"), (8192, 500, 768, "f32")])
def test_the_same_bits_every_time(dev, M, N, K, t):
    x, w = torch.randn(M, K, device=dev).to(TYPES[t]), hip.quant_fp8(torch.randn(N, K, device=dev))
    first = hip.linear_fp8(x, w, act="tanh")
    for _ in range(4):
        assert torch.equal(hip.linear_fp8(x, w, act="tanh"), first)
