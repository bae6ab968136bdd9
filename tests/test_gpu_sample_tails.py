"""GPU: cube_sample_rows on rows whose tail is flat: one hot logit over a background of one value or a few.  There the roundings of the
weights do not cancel, so this is where the running sum's own precision shows.

The borders are computed in integers: a weight is exp((z - max) / T) to 40 digits, times 2^200.  A row of V logits is off from them by
less than V * 2^-62 of the largest weight (each weight is cut to a whole 2^-62) and 2^-48 of itself (the exponential's own error, 2^-50,
on either side of the quotient), and u * total by 2^-52.  Each u lies in the middle of its token's share, which is more than four times
all of that wide: the tokens are compared for equality.  prob: one fp32 rounding (2^-24 of itself) and those errors, in all below
2^-23."""
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

from cube_amd import hip

pytestmark = pytest.mark.gpu
getcontext().prec = 60

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda", 0)


def weight(z, top, T=1.0):
    return int((Decimal(z - top) / Decimal(T)).exp() * 2 ** 200)


def expected(z, ranks):
    """z: one row as float64; ranks: places in the order -> (tokens, u in the middle of each token's share, their prob)."""
    order = np.argsort(-z, kind="stable")
    vals, count = np.unique(-z, return_counts=True)
    vals = -vals
    w = [weight(float(v), float(vals[0])) for v in vals]
    first = np.concatenate([[0], np.cumsum(count)])
    before = [0]
    for n, x in zip(count, w):
        before.append(before[-1] + int(n) * x)
    total = before[-1]
    u, p = [], []
    for r in ranks:
        g = int(np.searchsorted(first, r, side="right")) - 1
        u.append((2 * (before[g] + (int(r) - int(first[g])) * w[g]) + w[g]) / (2 * total))
        p.append(w[g] / total)
        err = len(z) * 2.0 ** -62 * 2.0 ** 200 / total + 2.0 ** -48 + 2.0 ** -52
        assert p[-1] > 8 * err, "the case itself is too fine"
    return order[ranks], np.array(u), np.array(p)


def background(V, hot, kind, t):
    z = np.zeros(V)
    if kind == "few":
        z[1::3], z[2::3] = 0.5, -0.25
    z[V // 3] = hot
    z = torch.from_numpy(z).to(TYPES[t])
    return z, z.double().numpy()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["flat", "few"])
@pytest.mark.parametrize("V,hot", [(300, 24.0), (5000, 20.75), (32003, 20.75), (32003, 25.0), (40000, 22.0), (250002, 20.75), (250002, 25.0), (1 << 22, 20.0)])
def test_one_hot_logit_over_a_flat_background(dev, V, hot, kind, t):
    z, zz = background(V, hot, kind, t)
    n = 96 if V < 1 << 20 else 24
    ranks = np.unique(np.concatenate([[0, 1, 2, V - 1, V - 2], np.linspace(1, V - 1, n).astype(np.int64)]))
    tok, u, p = expected(zz, ranks)
    rows = z.to(dev)[None].expand(len(ranks), V).contiguous()
    for M in (len(ranks), 1):                # (the form of a call may depend on the number of rows)
        got, prob = hip.sample_rows(rows[-M:], torch.from_numpy(u[-M:]).to(dev))
        np.testing.assert_array_equal(got.cpu().numpy(), tok[-M:])
        np.testing.assert_allclose(prob.cpu().double().numpy(), p[-M:], rtol=2.0 ** -23)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [5000, 40000, 1 << 22])
def test_a_tail_far_below_is_counted_as_it_is(dev, V, t):
    """A flat tail 28.5 nats below: at 2^22 logits it holds 1.7e-6 of the mass, and prob of the hot logit says so."""
    z, zz = background(V, 28.5, "flat", t)
    w = weight(0.0, float(zz.max()))
    total = 2 ** 200 + (V - 1) * w
    got, prob = hip.sample_rows(z.to(dev)[None], torch.zeros(1, dtype=torch.float64, device=dev))
    assert got.tolist() == [V // 3] and abs(prob.item() - 2 ** 200 / total) <= 2.0 ** -23
    # a tenth into the tail, and nine tenths: within the 2^-40 that the cut weights may move the border, of a token's 2^-41
    for part in (0.1, 0.9):
        u = (2 ** 200 + int(part * (V - 1)) * w) / total
        got, _ = hip.sample_rows(z.to(dev)[None], torch.full((1,), u, dtype=torch.float64, device=dev))
        place = got.item() - (1 if got.item() > V // 3 else 0)
        assert abs(place - int(part * (V - 1))) <= 2 + (V * 2.0 ** -62 + 2.0 ** -48 + 2.0 ** -52) * 2.0 ** 200 / w


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [5000, 40000, 250002])
def test_filters_that_end_inside_a_flat_tail(dev, V, t):
    """top-p whose border lies among equal logits, top-k there, min-p below them: the kept set ends where the integers say."""
    hot = 20.75
    z, zz = background(V, hot, "flat", t)
    w, top = weight(0.0, hot), 2 ** 200
    n = 1000                                                  # tail logits that stay
    row = z.to(dev)[None]
    last = n if n <= V // 3 else n + 1
    u = torch.tensor([1.0 - 2.0 ** -53], dtype=torch.float64, device=dev)
    tok, prob = hip.sample_rows(row, u, top_k=n + 1)
    assert tok.item() == last - 1 and abs(prob.item() - w / (top + n * w)) <= 2.0 ** -23 * w / (top + n * w)
    tok, _ = hip.sample_rows(row, u, min_p=float(np.float32(0.5 * w / top)))
    assert tok.item() == V - 1
    # p as fp32 comes in steps of 2^-24 of the total, some thousand tail logits: the border is computed from the rounded p
    total = top + (V - 1) * w
    p = np.float32((top + 0.4 * (V - 1) * w) / total)
    if p < 1:
        goal = int(Decimal(float(p)) * total)
        stay = -(-(goal - top) // w) if goal > top else 0
        tok, prob = hip.sample_rows(row, u, top_p=float(p))
        at = tok.item() + (0 if tok.item() > V // 3 else 1)
        at = 0 if tok.item() == V // 3 else at                # tail logits kept
        slack = 1 + (V * 2.0 ** -62 + 2.0 ** -48 + 2.0 ** -52) * top / w
        assert abs(at - stay) <= slack, (at, stay, slack)
