"""CPU: where a decoder's random numbers come from (networks/sampling.py)."""
import torch

from cube_amd.networks.sampling import Sampling


def test_every_start_gives_the_seeds_numbers():
    s = Sampling(temperature=0.7, top_k=4, top_p=0.9, min_p=0.1, seed=5)
    first = s.begin()
    a = [first.uniforms(8, 3, "cpu") for _ in range(2)]
    for _ in range(2):
        again = s.begin()
        assert (again.temperature, again.top_k, again.top_p, again.min_p, again.seed) == (0.7, 4, 0.9, 0.1, 5)
        b = [again.uniforms(8, 3, "cpu") for _ in range(2)]
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(b[0], b[1])
    other = Sampling(seed=6).begin().uniforms(8, 3, "cpu")
    assert not torch.equal(other, a[0])


def test_without_a_seed_every_start_goes_on():
    s = Sampling()
    assert not torch.equal(s.begin().uniforms(8, 3, "cpu"), s.begin().uniforms(8, 3, "cpu"))
