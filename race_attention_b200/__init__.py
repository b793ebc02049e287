"""B200-native (sm_100a) RACE attention: drop-in for the reference's
BatchedACE / RACEAttention / RACEBlock modules.

    from race_attention_b200 import race_attention          # autograd op
    from race_attention_b200.vit import RACEAttention        # non-causal
    from race_attention_b200.race import RACEAttention       # causal
    from race_attention_b200.fp8 import fp8_linear, rms_norm  # 8-bit layers around it
    from race_attention_b200.optim import AdamW               # states in 8 or 32 bits
"""
from .functional import race_attention  # noqa: F401

__all__ = ["race_attention"]
