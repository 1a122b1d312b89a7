"""trit_b200: the greedy token loop of Trit's decoder language model
(CausalLm) on NVIDIA B200, behind the C ABI of include/trit_cuda.h."""
from .lm import CausalLm, Dense, KvCache, Prefix, Rotary, TritError, library, rms_norm  # noqa: F401

__all__ = ["CausalLm", "Dense", "KvCache", "Prefix", "Rotary", "TritError", "library", "rms_norm"]
