"""User-facing configuration of a search over beams."""

from __future__ import annotations

from dataclasses import dataclass


@dataclass(frozen=True, slots=True)
class BeamSearchParams:
    """Parameters of one search (``LLM.beam_search``).

    Attributes:
        beam_width: continuations of a prompt that are followed at a time, and hypotheses returned.
        max_new_tokens: hard cap on the number of generated tokens.
        length_penalty: a hypothesis of ``n`` tokens is ranked by its sum of log probabilities over ``n **
            length_penalty``; 0 ranks by the sum, larger values favour longer ones.
        early_stopping: end a search as soon as it has ``beam_width`` ended hypotheses; otherwise it goes on until no
            running beam, were it to end now, would be ranked among them.
        ignore_eos: keep extending past EOS until the cap on tokens.
    """

    beam_width: int = 4
    max_new_tokens: int = 128
    length_penalty: float = 1.0
    early_stopping: bool = False
    ignore_eos: bool = False

    def __post_init__(self) -> None:
        if not 1 <= self.beam_width <= 32:
            raise ValueError(f"beam_width must be in [1, 32], got {self.beam_width}")
        if self.max_new_tokens < 1:
            raise ValueError(f"max_new_tokens must be >= 1, got {self.max_new_tokens}")
        if not self.length_penalty >= 0.0:
            raise ValueError(f"length_penalty must be >= 0, got {self.length_penalty}")
