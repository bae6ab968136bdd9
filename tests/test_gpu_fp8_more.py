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
