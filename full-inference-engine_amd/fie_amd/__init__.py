"""MI355X-native fused token sampler with the reference engine's sampler surface.

``fie_amd.batching.sampler.BatchedSampler`` and ``fie_amd.runtime.sampling`` mirror
``engine.batching.sampler`` and ``engine.runtime.sampling`` of full-inference-engine.
Beside them: ``fie_amd.verify`` (drafted tokens), ``fie_amd.linear`` (products in 8-bit
integers), ``fie_amd.norm`` (block norms), ``fie_amd.beam`` (beam search), ``fie_amd.pages`` (pages of a
cache) and ``fie_amd.adapters`` (low-rank adapters).
"""

from .batching.sampler import BatchedSampler, SampleResult, VerifyResult
from .beam import BeamSearch
from .runtime.sampling import GREEDY, SamplingParams

__all__ = ["BatchedSampler", "BeamSearch", "SampleResult", "VerifyResult", "SamplingParams", "GREEDY"]
