"""GPU: the framework's own paths through the 8-bit Linear layers and the sampler: an LM encoder with Fp8Linear layers behind LMHelperHF
(networks/fp8.py, networks/lm.py), and the lemmatizer's decoder with drawn characters (networks/sampling.py)."""
import numpy as np
import pytest
import torch

from cube_amd import hip
from oracle import ops_oracle as oo
from tests import cases
from tests.test_gpu_fp8 import close, np_

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


def check_linear(x, y, weight, bias):
    """One call of an Fp8Linear: what went in, what came out, the float layer it stands for."""
    x, y = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
    a, w = oo.rows_value(*oo.quant(np_(x))), oo.rows_value(*oo.quant(np_(weight)))
    want, mag = oo.gemm(a, w, None if bias is None else np_(bias.float()))
    close(np_(y), want, mag, x.shape[1], {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[y.dtype])


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("lead", [(), (1,), (7,), (2, 40), (3, 5, 20)])
def test_fp8_linear(dev, t, bias, lead):
    from cube_amd.networks.fp8 import Fp8Linear
    torch.manual_seed(len(lead))
    lin = torch.nn.Linear(300, 170, bias=bias).to(dev)
    f = Fp8Linear(lin)
    x = torch.randn(*lead, 300, device=dev).to(t)
    with torch.no_grad():
        y = f(x)
    assert y.shape == lead + (170,) and y.dtype == t
    check_linear(x, y, lin.weight, lin.bias)


def test_fp8_linear_as_a_module(dev):
    """Moves, type changes, its state dict, inputs that are not contiguous, and the refusal to train."""
    from cube_amd.networks.fp8 import Fp8Linear, quantise_linears
    lin = torch.nn.Linear(200, 30).to(dev)
    f = Fp8Linear(lin)
    x = torch.randn(6, 200, device=dev)
    with torch.no_grad():
        y = f(x)
        f.half()
        assert f.bias.dtype == torch.float32 and torch.equal(f(x), y)
        f.to("cpu")
        with pytest.raises(ValueError):
            f(x)
        f.to(dev)
        assert torch.equal(f(x), y)
        other = Fp8Linear(torch.nn.Linear(200, 30).to(dev))
        other.load_state_dict(f.state_dict())
        assert torch.equal(other(x), y)
        wide = torch.randn(6, 400, device=dev)
        wide[:, 100:300] = x
        assert torch.equal(f(wide[:, 100:300]), y)
        cols = torch.randn(200, 6, device=dev)
        cols.copy_(x.t())
        assert torch.equal(f(cols.t()), y)
        assert torch.equal(f(x[:1].expand(6, 200)), y[:1].expand(6, 30)) and f(x[:0]).shape == (0, 30)
    with pytest.raises(ValueError, match="gradient"):
        f(x.clone().requires_grad_())
    net = torch.nn.Sequential(torch.nn.Linear(8, 8), torch.nn.ModuleList([torch.nn.Linear(8, 4), torch.nn.LayerNorm(4)])).to(dev)
    assert quantise_linears(net) == 2 and not any(type(m) is torch.nn.Linear for m in net.modules())


def test_lm_helper_with_an_8_bit_encoder(dev):
    """LMHelperHF(fp8=True) over a small transformer: every Linear call inside is the product of the quantised operands, and what `apply`
    fills in is the pooling of those hidden states."""
    transformers = pytest.importorskip("transformers")
    from cube_amd.networks.fp8 import Fp8Linear
    from cube_amd.networks.lm import LMHelperHF
    torch.manual_seed(5)
    cfg = transformers.XLMRobertaConfig(vocab_size=cases.LM_PIECES, hidden_size=96, num_hidden_layers=2, num_attention_heads=4,
                                        intermediate_size=200, max_position_embeddings=520, output_hidden_states=True)
    enc = transformers.XLMRobertaModel(cfg)
    weights = {n: (m.weight.detach().clone(), m.bias.detach().clone()) for n, m in enc.named_modules() if type(m) is torch.nn.Linear}
    h = LMHelperHF(device=dev, splitter=cases.FakeSplitter(), encoder=enc, fp8=True)
    names = {m: n for n, m in enc.named_modules() if type(m) is Fp8Linear}
    assert sorted(names.values()) == sorted(weights) and not any(type(m) is torch.nn.Linear for m in enc.modules())
    seen = []
    for m in names:
        m.register_forward_hook(lambda mod, args, out: seen.append((names[mod], args[0].clone(), out.clone())))
    _, penc, _ = cases.parser_model(cases.FULL)
    doc = cases.lm_document(penc)
    doc.sentences = doc.sentences[:3]
    h.apply(doc)
    assert len(seen) >= 3 * len(names) - 3      # (the pooler may not run)
    for n, x, y in seen:
        check_linear(x, y, *weights[n])
    for s in doc.sentences:
        for w in s.words:
            assert len(w.emb) == 3 and all(v.shape == (96,) and np.isfinite(v).all() for v in w.emb)


# ---- the lemmatizer's decoder -----------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lemma(dev):
    from cube_amd.networks.lemmatizer import LemmaDataset, Lemmatizer, Word2TargetCollate
    cfg, enc, sd = cases.lemmatizer_model(cases.LEMMA_SMALL)
    m = Lemmatizer(cfg, enc)
    m.load_state_dict(sd)
    m.to(dev)
    ds = LemmaDataset(cases.lemma_document(enc, "ragged"), for_training=False)
    X = Word2TargetCollate(enc).collate_fn([ds[i] for i in range(len(ds))], targets=False)
    return m, enc, X


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=5), dict(top_p=0.8), dict(temperature=1.3, min_p=0.1, top_k=20, top_p=0.95)])
@pytest.mark.parametrize("fused", [True, False])
def test_drawn_characters_are_the_oracles(lemma, kw, fused):
    """Each step's characters are what the oracle draws from that step's logits and random numbers (the end symbol among the
    candidates, the start symbol behind it not), and the fed-back state goes on from them."""
    from cube_amd.networks.sampling import Sampling
    m, enc, X = lemma
    m.fused_cell = fused
    try:
        ed = m._encode(X)
        oc, ok, n, logits = m._decode(ed, max_steps=19, keep_logits=True, sampling=Sampling(seed=3, **kw))
    finally:
        del m.fused_cell
    u = torch.cat(ed["uniforms"]).cpu().numpy()
    z = logits.cpu().double().numpy()
    V = len(enc.char2int) + 1
    T, p, mp = (float(np.float32(kw.get(k, d))) for k, d in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0)))
    assert oc.max() < V and n > 0
    near = 0
    for s in range(n):
        for b in range(oc.shape[0]):
            et, _, d = oo.sample_row(z[s, b, :V], u[s, b], T, kw.get("top_k", 0), p, mp)
            near += et != oc[b, s] and d < 2.0 ** -36
            assert et == oc[b, s] or d < 2.0 ** -36, (s, b)
    assert near <= 1


def test_temperature_zero_is_the_greedy_decoder(lemma):
    from cube_amd.networks.sampling import Sampling
    m, enc, X = lemma
    m.max_steps = 24
    try:
        a, b = m.decode_batch(X), m.decode_batch(X, sampling=Sampling(temperature=0.0))
        if (a[0] <= len(enc.char2int)).all():       # (the greedy decoder may emit the start symbol, the drawn one may not)
            np.testing.assert_array_equal(a[0], b[0])
            np.testing.assert_array_equal(a[1], b[1])
        one, two, other = (m.decode_batch(X, sampling=Sampling(seed=s)) for s in (11, 11, 12))
        np.testing.assert_array_equal(one[0], two[0])
        assert one[0].shape != other[0].shape or (one[0] != other[0]).any()
        np.testing.assert_array_equal(m.decode_batch(X)[0], a[0])      # the greedy decoder afterwards is what it was
    finally:
        m.max_steps = None


def test_process_draws_lemmas(lemma):
    """Lemmatizer.process(sampling=...) fills every word; the same seed gives the same document."""
    from cube_amd.networks.lemmatizer import Word2TargetCollate
    from cube_amd.networks.sampling import Sampling
    m, enc, _ = lemma
    m.max_steps = 16
    try:
        out = []
        for seed in (1, 1, 2):
            doc = cases.lemma_document(enc, "ragged")
            m.process(doc, Word2TargetCollate(enc), batch_size=8, num_workers=0, sampling=Sampling(temperature=0.9, top_p=0.95, seed=seed))
            out.append([w.lemma for s in doc.sentences for w in s.words])
        assert out[0] == out[1] != out[2] and all(isinstance(x, str) for x in out[0])
    finally:
        m.max_steps = None


@pytest.mark.parametrize("bad", [dict(temperature=-1), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2.5), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2)])
def test_sampling_refuses(bad):
    from cube_amd.networks.sampling import Sampling
    with pytest.raises(ValueError):
        Sampling(**bad)
