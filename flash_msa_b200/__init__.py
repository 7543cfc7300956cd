"""flash_msa_b200: the Flash-MSA training hot path on B200 (sm_100a).

Public names are those of the reference package (flash_msa/__init__.py:3-14)."""
from .api import sparse_attention as flash_msa_func
from .api import sparse_attention_varlen as flash_msa_varlen_func
from .api import sparse_attention_warmup
from .api import sparse_attention_warmup_varlen as flash_msa_warmup_varlen_func
from .api import sparse_attention_warmup as flash_msa_func_warmup
from .api import sparse_attention_warmup as flash_msa_warmup_func
from .api import check_pending_status, last_kl_value
from .serving import cache_append as flash_msa_cache_append
from .serving import cache_attention as flash_msa_cache_func
from .serving import cache_empty as flash_msa_cache_empty
from .serving import cache_evict as flash_msa_cache_evict
from .serving import cache_unpack as flash_msa_cache_unpack
from .serving import prompt_attention as flash_msa_prompt_func

__all__ = [
    "flash_msa_func",
    "flash_msa_varlen_func",
    "flash_msa_warmup_varlen_func",
    "flash_msa_func_warmup",
    "flash_msa_warmup_func",
    "sparse_attention_warmup",
    "last_kl_value",
    "check_pending_status",
    "flash_msa_cache_append",
    "flash_msa_cache_empty",
    "flash_msa_cache_evict",
    "flash_msa_cache_func",
    "flash_msa_cache_unpack",
    "flash_msa_prompt_func",
]
