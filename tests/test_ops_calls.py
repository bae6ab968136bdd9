"""CPU: what the calls on tensors of the 8-bit Linear operators and the sampler (cube_amd/hip.py) refuse before anything is launched."""
import pytest
import torch
from torch.autograd import forward_ad

from cube_amd import hip


def rows(n=4, columns=200):
    return hip.Fp8Rows(torch.zeros(n, 256, dtype=torch.uint8), torch.zeros(1, n, dtype=torch.int32), columns)


def f64(n=4):
    return torch.full((n,), 0.5, dtype=torch.float64)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(grad):
    """A dual tensor does not require a gradient, and no_grad() does not turn its tangent off: it would be lost without a word."""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x = forward_ad.make_dual(torch.randn(4, 200), torch.randn(4, 200))
        for call in (lambda: hip.quant_fp8(x), lambda: hip.linear_fp8(x, rows()), lambda: hip.sample_rows(x, f64())):
            with pytest.raises(ValueError, match="tangent"):
                call()
        v = forward_ad.make_dual(torch.randn(4), torch.randn(4))
        with pytest.raises(ValueError, match="tangent"):
            hip._vector("linear_fp8", "bias", v, 4, torch.float32, v.device)
        with pytest.raises(hip.CubeHipError, match="no CPU fallback"):    # without a tangent: the next refusal
            hip.quant_fp8(torch.randn(4, 200))
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.quant_fp8(torch.randn(4, 200))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_vectors_that_ask_for_a_gradient_are_refused(dtype):
    """bias, u, and the settings of a draw (a temperature that is learnt): refused unless gradients are off."""
    v = torch.full((4,), 0.7, dtype=dtype, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        hip._vector("sample_rows", "temperature", v, 4, dtype, v.device)
    with torch.no_grad():
        assert hip._vector("sample_rows", "temperature", v, 4, dtype, v.device) == v.data_ptr()
    assert hip._vector("sample_rows", "temperature", v.detach(), 4, dtype, v.device) == v.data_ptr()


def test_negated_views_are_refused():
    """The imaginary part of a conjugate is its memory with the sign changed: one column (or value) of it passes as neighbouring ones."""
    x = torch.zeros(4, 1, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    for call in (lambda: hip.quant_fp8(x), lambda: hip.sample_rows(x, f64()), lambda: hip._vector("linear_fp8", "bias", x[:1, 0], 1, torch.float32, x.device)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.quant_fp8(x.resolve_neg())


@pytest.mark.parametrize("shape", [(1 << 31, 2), ((1 << 32) + 4, 2), (1, 1 << 31), (2, (1 << 32) + 100)])
def test_sizes_beyond_31_bits_are_refused(shape):
    """The C functions take 32-bit counts, and ctypes drops what is above them: 2^32 + 100 columns were 100."""
    x = torch.zeros(1, 1).expand(shape)
    for call in (lambda: hip.quant_fp8(x), lambda: hip.linear_fp8(x, rows()), lambda: hip.sample_rows(x, f64())):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    if shape[1] == 2:
        with pytest.raises(ValueError, match="2\\^31"):
            hip.Fp8Rows(torch.zeros(1, 1, dtype=torch.uint8).expand(shape[0], 128), torch.zeros(1, 1, dtype=torch.int32).expand(1, shape[0]), 100)
    else:
        with pytest.raises(ValueError, match="2\\^31"):
            hip.Fp8Rows(torch.zeros(1, 128, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32), shape[1])
