"""B200-native shared-prefix paged attention: the hot path of ParrotServe's builtin engine.

Public surface mirrors ``parrot/engine/builtin/kernels/__init__.py:7-16``.
"""
from .ops import (  # noqa: F401
    AttentionCall,
    HostStep,
    HostStepPipeline,
    discontinuous_move_tokens,
    flash_paged_attention,
    flash_paged_attention_grouped,
    gather_cached_kv,
    move_tokens_from_blocked_k_cache,
    move_tokens_from_blocked_v_cache,
    paged_flash_attention,
    rotary_reshape_and_cache,
    sample_top_p,
    vllm_paged_attention,
    vllm_reshape_and_cache,
    vllm_rotary_emb,
)
from .fp8 import (  # noqa: F401
    Fp8AttentionCall,
    fp8_flash_paged_attention,
    fp8_flash_paged_attention_grouped,
    fp8_gather_cached_kv,
    fp8_kv_cache,
    fp8_paged_attention,
    fp8_reshape_and_cache,
)
from .tables import BlockTables, build_block_tables  # noqa: F401
from . import attention_ops, cache_ops  # noqa: F401
from .sampler import Sampler  # noqa: F401

__version__ = "0.1.0"
