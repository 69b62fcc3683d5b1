from .layer import MuZeroCacheLayer
from .paged import MuZeroPagedCache
from .attention import mu_zero_decode_attention_forward

__all__ = ["MuZeroCacheLayer", "MuZeroPagedCache", "mu_zero_decode_attention_forward"]
