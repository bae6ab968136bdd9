"""GPU: cube_sample_rows, calls that the other files of this operator do not make."""
import numpy as np
import pytest
import torch

from cube_amd import hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V", [(70, 17000), (300, 33000), (40, 70000), (3, 70000)])
def test_greedy_rows_of_every_long_form(dev, M, V, t):
    """The arg-max of rows whose largest value lies in any octave of either sign, or twice: the first of them, every time."""
    g = torch.Generator().manual_seed(M + V)
    z = torch.randn(M, V, generator=g) * torch.exp2(torch.randint(-12, 6, (M, 1), generator=g).float())
    z[::3] -= 40.0 * torch.rand(len(z[::3]), 1, generator=g) + z[::3].max(1, keepdim=True).values   # all negative
    z = z.to(TYPES[t])
    want = z.double().numpy().argmax(1)
    u = torch.full((M,), 0.5, dtype=torch.float64, device=dev)
    for _ in range(3):
        tok, prob = hip.sample_rows(z.to(dev), u, temperature=0.0)
        np.testing.assert_array_equal(tok.cpu().numpy(), want)
        assert bool((prob == 1).all())


def test_settings_that_ask_for_a_gradient(dev):
    z, u = torch.randn(4, 60, device=dev), torch.full((4,), 0.5, dtype=torch.float64, device=dev)
    for name in ("temperature", "top_p", "min_p"):
        v = torch.full((4,), 0.7, device=dev, requires_grad=True)
        with pytest.raises(ValueError, match="gradient"):
            hip.sample_rows(z, u, **{name: v})
        with torch.no_grad():
            got = hip.sample_rows(z, u, **{name: v})
        assert torch.equal(got[0], hip.sample_rows(z, u, **{name: v.detach()})[0])
    with pytest.raises(ValueError, match="gradient"):
        hip.sample_rows(z, u.clone().requires_grad_())
