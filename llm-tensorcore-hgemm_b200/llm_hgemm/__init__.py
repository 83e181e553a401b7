"""B200 (sm_100a) FP16 HGEMM for LLM linear layers.

Drop-in for the reference package of the same name
(reference llm_hgemm/__init__.py:3-5): ``hgemm`` and ``available_providers``.
Importing it loads the native extension and fails loudly when it is missing.
Training operators (no reference counterpart): ``gated_ffn``,
``linear_cross_entropy`` and ``orthogonalize``.
"""

from .ops import available_providers, hgemm
from .training import gated_ffn, linear_cross_entropy, orthogonalize

__all__ = ["available_providers", "gated_ffn", "hgemm", "linear_cross_entropy", "orthogonalize"]
