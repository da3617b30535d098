"""What a request asks of the sampler."""

from __future__ import annotations

import math
from dataclasses import dataclass


@dataclass
class SamplingParams:
    """Names and meanings after the reference's generate() (serving/executor.py:334-345)
    and its dev command line (serving/cli.py:18-23): ``max_new`` tokens at most;
    ``temperature`` <= 0 is greedy (the engine facade's default, serving/executor.py:539);
    ``top_k``/``top_p`` filter as runtime/sampler.py:60-79 does; ``seed`` seeds the
    request's own generator; ``repetition_penalty`` as runtime/sampler.py:12-33;
    a token in ``stop_ids`` ends the request and is not part of its output."""
    max_new: int = 16
    temperature: float = 0.0
    top_k: int | None = None
    top_p: float | None = None
    seed: int | None = None
    repetition_penalty: float | None = None
    stop_ids: tuple = ()

    def __post_init__(self):
        if self.max_new < 1:
            raise ValueError("max_new must be >= 1")
        if self.top_k is not None and int(self.top_k) <= 0:
            raise ValueError("top_k must be >= 1")          # runtime/sampler.py:62-63
        self.stop_ids = tuple(int(s) for s in self.stop_ids)

    @property
    def penalised(self) -> bool:
        """Whether a repetition penalty applies (runtime/sampler.py:24: none, <= 0 and 1 change nothing)."""
        p = self.repetition_penalty
        return p is not None and p > 0 and p != 1.0


@dataclass
class BeamParams:
    """What a request asks of a beam search (the reference has none).  ``beams`` continuations are kept alive; a continuation ends with a token of
    ``stop_ids`` (not part of its output) or at ``max_new`` tokens; finished ones are ranked by cumulative log-probability over
    ``n ** length_penalty``, n their tokens with the stop; the ``results`` best come back (None: as many as beams).  The search ends when no living continuation could
    still get among them, so that its results are those of a search to the last token."""
    beams: int = 4
    max_new: int = 16
    length_penalty: float = 1.0
    stop_ids: tuple = ()
    results: int | None = None

    def __post_init__(self):
        self.stop_ids = tuple(sorted({int(s) for s in self.stop_ids}))
        if self.results is None:
            self.results = self.beams
        if not 1 <= self.beams <= 32 or not 1 <= self.results <= 32:
            raise ValueError("beams and results are 1 to 32")
        if self.max_new < 1:
            raise ValueError("max_new must be >= 1")
        if not abs(self.length_penalty) < 64:
            raise ValueError("length_penalty must be between -64 and 64")
        if abs(self.length_penalty) * math.log2(self.max_new) > 64:
            raise ValueError(f"length_penalty {self.length_penalty} at {self.max_new} tokens: the scores of finished continuations would leave float32 (max_new ** length_penalty is within 2^-64 and 2^64)")
        if self.keep > 128:
            raise ValueError(f"{self.beams} beams with {len(self.stop_ids)} stop ids need {self.keep} candidates a step, 128 at most")

    @property
    def keep(self) -> int:
        """Candidates a step: every beam may lose one to each stop id, and as many as there are beams have to go on."""
        return self.beams * (1 + len(self.stop_ids))
