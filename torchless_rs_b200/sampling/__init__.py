from .params import SamplingParams, uniform_for

__all__ = ["SamplingParams", "uniform_for", "Sampler", "BeamSelector"]


def __getattr__(name):
    if name == "Sampler":
        from .sampler import Sampler
        return Sampler
    if name == "BeamSelector":
        from .beam import BeamSelector
        return BeamSelector
    raise AttributeError(name)
