"""Per-request sampling parameters."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional


@dataclass(frozen=True)
class SamplingParams:
    """temperature 0 is greedy (the reference's only mode, src/csrc/model/gpt/gpt.cc:628-636);
    a positive temperature samples softmax(logits / temperature) with noise that depends
    only on (seed, index of the output token).  Of a positive temperature's distribution ``top_k`` (0: all) keeps the most
    likely tokens, ``top_p`` (1: all) the fewest of those that hold so much of their probability, ``min_p`` (0: all) the ones with so
    much of the likeliest one's; a request with any of them draws by one random number a token, from (seed, index) too.
    Generation ends at ``max_new_tokens``
    (the reference's MAX_DECODING_STEP, src/examples/run_gpt.cc:24), at the end token
    unless ``ignore_eos`` (src/examples/lib/inference_batch.cc:199-201), or when the
    model's positions are used up."""
    temperature: float = 0.0
    max_new_tokens: int = 128
    seed: int = 0
    eos_token_id: Optional[int] = None     # None: the model's own
    ignore_eos: bool = False
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    @property
    def filtered(self) -> bool:
        """Whether any filter narrows the choice."""
        return self.temperature > 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0)

    def __post_init__(self):
        if self.top_k < 0:
            raise ValueError("top_k must be >= 0")
        if not 0 < self.top_p <= 1:
            raise ValueError("top_p must be in (0, 1]")
        if not 0 <= self.min_p <= 1:
            raise ValueError("min_p must be in [0, 1]")
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if self.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be >= 1")
