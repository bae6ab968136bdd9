"""GPU: one Sampling object used for several calls of the lemmatizer."""
import numpy as np
import pytest
import torch

from tests import cases
from tests.test_gpu_fp8_sampling_paths import dev, lemma  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def test_one_object_draws_the_same_every_time(lemma):
    """decode_batch and process twice with one seeded object, other calls between: the same characters and lemmas.  Without a seed a
    second call draws others."""
    from cube_amd.networks.lemmatizer import Word2TargetCollate
    from cube_amd.networks.sampling import Sampling
    m, enc, X = lemma
    m.max_steps = 16
    try:
        s, free = Sampling(temperature=0.9, seed=4), Sampling(temperature=0.9)
        out = []
        for _ in range(2):
            chars, _ = m.decode_batch(X, sampling=s)
            doc = cases.lemma_document(enc, "ragged")
            m.process(doc, Word2TargetCollate(enc), batch_size=8, num_workers=0, sampling=s)
            out.append((chars, [w.lemma for t in doc.sentences for w in t.words]))
        np.testing.assert_array_equal(out[0][0], out[1][0])
        assert out[0][1] == out[1][1]
        a, b = (m.decode_batch(X, sampling=free)[0] for _ in range(2))
        assert a.shape != b.shape or (a != b).any()
    finally:
        m.max_steps = None
    assert torch.cuda.is_available()
