from .sampling_params import BeamSearchParams, InvalidRequest, JitableSamplingParams, SamplingParams

__all__ = ["SamplingParams", "InvalidRequest", "JitableSamplingParams", "BeamSearchParams"]
