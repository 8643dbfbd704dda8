from .controls import ControlTable, RequestControls
from .sampler import Sampler, SamplingRow

__all__ = ["ControlTable", "RequestControls", "Sampler", "SamplingRow"]
