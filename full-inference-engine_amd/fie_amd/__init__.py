"""MI355X-native fused token sampler with the reference engine's sampler surface.

``fie_amd.batching.sampler.BatchedSampler`` and ``fie_amd.runtime.sampling`` mirror
``engine.batching.sampler`` and ``engine.runtime.sampling`` of full-inference-engine.
Beside them: ``fie_amd.verify`` (drafted tokens), ``fie_amd.linear`` (products in 8-bit
integers) and ``fie_amd.norm`` (block norms).
"""

from .batching.sampler import BatchedSampler, SampleResult, VerifyResult
from .runtime.sampling import GREEDY, SamplingParams

__all__ = ["BatchedSampler", "SampleResult", "VerifyResult", "SamplingParams", "GREEDY"]
