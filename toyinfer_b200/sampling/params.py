"""Sampling options, with the reference's names, meanings and defaults
(include/options.h:17-20, src/options.cpp:33-35)."""
from __future__ import annotations

from dataclasses import dataclass


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.6
    top_k: int = 20          # 0 or >= vocabulary: no limit
    top_p: float = 0.95      # 1.0: no limit
    seed: int = 0

    @property
    def greedy(self) -> bool:
        """The reference's rule (src/sampler.cpp:20): argmax when the temperature is
        (nearly) zero or only one candidate may be kept."""
        return abs(self.temperature) < 1e-3 or self.top_k == 1

    def check(self) -> None:
        if self.temperature < 0:
            raise ValueError(f"temperature must not be negative, got {self.temperature}")
        if not (0.0 < self.top_p <= 1.0):
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if self.top_k < 0:
            raise ValueError(f"top_k must not be negative, got {self.top_k}")


GREEDY = SamplingParams(temperature=0.0, top_k=1, top_p=1.0)


@dataclass(frozen=True)
class BeamParams:
    """Options of beam search, with the reference's --beam_size and --length_penalty (include/options.h, src/options.cpp).

    A hypothesis's value is its score (the sum of its tokens' log-probabilities, the stop token's among them) divided by
    the number of its drawn tokens to the power of ``length_penalty``.  A search ends when it holds ``beams`` ended
    hypotheses and no running one can come to a better value than the worst of them, or with ``early_stopping`` as soon
    as it holds them."""

    beams: int = 4
    length_penalty: float = 1.0
    early_stopping: bool = False
    n_best: int = 1              # hypotheses returned per request, best first

    def check(self) -> None:
        from ..kernels.beam import BEAMS_MAX
        if not 1 <= self.beams <= BEAMS_MAX:
            raise ValueError(f"beams must be between 1 and {BEAMS_MAX}, got {self.beams}")
        if not 0.0 <= self.length_penalty <= 5.0:
            raise ValueError(f"length_penalty must be between 0 and 5, got {self.length_penalty}")
        if not 1 <= self.n_best <= self.beams:
            raise ValueError(f"n_best must be between 1 and beams, got {self.n_best}")
