from .beam import BeamSearchParams
from .params import SamplingParams

__all__ = ["BeamSearchParams", "SamplingParams"]
