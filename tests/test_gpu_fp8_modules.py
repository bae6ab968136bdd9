"""GPU: Fp8Linear (networks/fp8.py) in modules that use their Linear layers in other ways than by calling them."""
import copy

import numpy as np
import pytest
import torch

from cube_amd import hip
from oracle import ops_oracle as oo
from tests.test_gpu_fp8 import np_
from tests.test_gpu_fp8_sampling_paths import check_linear

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


def converted(net):
    """-> (net with 8-bit layers, {layer: (name, weight, bias) of the Linear it stands for})"""
    from cube_amd.networks.fp8 import Fp8Linear, quantise_linears
    was = {n: (m.weight.detach().clone(), None if m.bias is None else m.bias.detach().clone()) for n, m in net.named_modules() if type(m) is torch.nn.Linear}
    quantise_linears(net)
    return {m: (n, *was[n]) for n, m in net.named_modules() if type(m) is Fp8Linear}


def run_and_check(net, layers, call):
    """The output of `call` without hooks on the layers and with them (torch's encoder layers take another way then): the same bits, and
    every layer's call is the product of its quantised operands."""
    with torch.no_grad():
        plain = call()
        seen = []
        hooks = [m.register_forward_hook(lambda mod, args, out: seen.append((mod, args[0].clone(), out.clone()))) for m in layers]
        again = call()
        for h in hooks:
            h.remove()
    assert torch.equal(plain, again) and {m for m, _, _ in seen} == set(layers)
    for m, x, y in seen:
        check_linear(x, y, *layers[m][1:])


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_torch_encoder_layers_in_evaluation(dev, t):
    torch.manual_seed(3)
    net = torch.nn.TransformerEncoder(torch.nn.TransformerEncoderLayer(64, 4, 160, batch_first=True), 2).to(dev).to(t).eval()
    x = torch.randn(3, 17, 64, device=dev).to(t)
    layers = converted(net)
    assert len(layers) == 4
    run_and_check(net, layers, lambda: net(x))
    pad = torch.zeros(3, 17, dtype=torch.bool, device=dev)
    pad[1, 9:] = True
    run_and_check(net, layers, lambda: net(x, src_key_padding_mask=pad))


def test_an_encoder_that_asks_for_a_weights_type(dev):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(4)
    net = transformers.T5EncoderModel(transformers.T5Config(vocab_size=90, d_model=64, d_kv=16, d_ff=128, num_layers=2, num_heads=4)).to(dev).eval()
    ids = torch.arange(40, device=dev).reshape(2, 20)
    layers = converted(net)
    assert layers
    run_and_check(net, layers, lambda: net(ids).last_hidden_state)


def test_the_weight_stands_for_the_rows(dev):
    from cube_amd.networks.fp8 import Fp8Linear
    lin = torch.nn.Linear(200, 30).to(dev)
    f = Fp8Linear(lin)
    want = oo.rows_value(*oo.quant(np_(lin.weight)))[:, :200]
    w = f.weight
    assert isinstance(w, torch.Tensor) and w.shape == (30, 200) and w.dtype == torch.float32 and w.device == lin.weight.device and not w.requires_grad
    np.testing.assert_array_equal(np_(w + 0), want)
    np.testing.assert_array_equal(np_(w.t()[3:5]), want.T[3:5])
    np.testing.assert_array_equal(np_(w.float()), want)
    x = torch.eye(200, device=dev)
    np.testing.assert_allclose(np_(torch.nn.functional.linear(x, w)), want.T, rtol=2.0 ** -22)
    with pytest.raises(ValueError, match="written"):
        w.mul_(2)
    with pytest.raises(hip.CubeHipError):
        hip.quant_fp8(w)
    f.half()
    assert f.weight.dtype == torch.float16 and "kind" not in f.state_dict()
    f.float()
    assert f.weight.dtype == torch.float32 and f.cpu().weight.device.type == "cpu"
    assert set(f.state_dict()) == {"q", "scale", "bias"}
    g = copy.deepcopy(f).to(dev)
    y = torch.randn(5, 200, device=dev)
    with torch.no_grad():
        assert torch.equal(g(y), f.to(dev)(y))


def test_the_buffers_are_what_counts(dev):
    """Buffers set by assignment, by a state dict that replaces them, and for one call by torch.func.functional_call."""
    from cube_amd.networks.fp8 import Fp8Linear
    torch.manual_seed(6)
    a, b = (Fp8Linear(torch.nn.Linear(200, 30).to(dev)) for _ in range(2))
    x = torch.randn(5, 200, device=dev)
    with torch.no_grad():
        ya, yb = a(x), b(x)
        assert not torch.equal(ya, yb)
        assert torch.equal(torch.func.functional_call(a, dict(b.named_buffers()), (x,)), yb) and torch.equal(a(x), ya)
        a.load_state_dict(b.state_dict(), assign=True)
        assert torch.equal(a(x), yb)
        c = Fp8Linear(torch.nn.Linear(200, 30).to(dev))
        c.q, c.scale, c.bias = b.q.clone(), b.scale.clone(), b.bias.clone()
        assert torch.equal(c(x), yb) and torch.equal(c.weight + 0, b.weight + 0)


def test_a_layer_in_several_places_stays_one(dev):
    """Under a second name of the same parent, and in another parent: one 8-bit layer, counted once; evaluation stays evaluation."""
    from cube_amd.networks.fp8 import Fp8Linear, quantise_linears

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Linear(16, 16)
            self.b = self.a
            self.c = torch.nn.Sequential(self.a, torch.nn.Linear(16, 4))

    net = Net().to(dev).eval()
    assert quantise_linears(net) == 2
    assert type(net.a) is Fp8Linear and net.b is net.a and net.c[0] is net.a and type(net.c[1]) is Fp8Linear
    assert not any(type(m) is torch.nn.Linear for m in net.modules()) and not any(m.training for m in net.modules())
    assert quantise_linears(net) == 0
