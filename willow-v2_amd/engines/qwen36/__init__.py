from .attention_hip import HipAttention, Rotary  # noqa: F401
from .moe_hip import HipMoE  # noqa: F401
