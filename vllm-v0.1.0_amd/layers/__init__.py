from .activation import SiluAndMul, get_act_fn  # noqa: F401
from .attention import PagedAttention, PagedAttentionWithRoPE  # noqa: F401
from .layernorm import RMSNorm  # noqa: F401
from .rotary import RotaryEmbedding, rotary_cos_sin_cache  # noqa: F401
