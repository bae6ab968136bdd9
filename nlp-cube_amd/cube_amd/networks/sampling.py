"""Sampled decoding: the settings of `cube_sample_rows` as a decoder takes them (no counterpart in the reference, whose decoder
is greedy, cube/networks/lemmatizer.py:160-167)."""
import copy

import torch


class Sampling:
    """temperature, top_k, top_p, min_p of a decoder's draws (numbers; include/cube_hip.h says what each keeps) and where their random
    numbers come from: `seed` (every call of process / decode_batch starts from it: the same draws every time for the same batches)
    or, where it is None, torch's own generator of the device."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed=None):
        if not temperature >= 0:
            raise ValueError("temperature must be 0 (greedy) or more, got %r" % (temperature,))
        if not (top_k >= 0 and top_k % 1 == 0):
            raise ValueError("top_k must be a whole number, 0 for no limit, got %r" % (top_k,))
        if not 0 <= top_p <= 1 or not 0 <= min_p <= 1:
            raise ValueError("top_p and min_p lie in 0..1, got %r, %r" % (top_p, min_p))
        self.temperature, self.top_k, self.top_p, self.min_p = float(temperature), int(top_k), float(top_p), float(min_p)
        self.seed = seed
        self._generators = {}

    def begin(self):
        """The same settings at the start of their random numbers: what one call of a decoder draws from."""
        s = copy.copy(self)
        s._generators = {}
        return s

    def uniforms(self, steps, rows, device):
        """float64 [steps, rows] in [0, 1) on the device."""
        g = None
        if self.seed is not None:
            g = self._generators.get(device)
            if g is None:
                g = self._generators[device] = torch.Generator(device=device).manual_seed(self.seed)
        return torch.rand((steps, rows), dtype=torch.float64, device=device, generator=g)
