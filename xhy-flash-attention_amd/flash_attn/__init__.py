"""MI355X-native FlashAttention-2 (drop-in for the reference ``flash_attn`` 2.0.8 API)."""
__version__ = "2.0.8"

from flash_attn.flash_attn_interface import flash_attn_func
from flash_attn.flash_attn_interface import flash_attn_kvpacked_func
from flash_attn.flash_attn_interface import flash_attn_qkvpacked_func
from flash_attn.flash_attn_interface import flash_attn_varlen_qkvpacked_func
from flash_attn.flash_attn_interface import flash_attn_varlen_kvpacked_func
from flash_attn.flash_attn_interface import flash_attn_varlen_func
from flash_attn.kvcache_interface import flash_attn_kvcache_commit_
from flash_attn.kvcache_interface import flash_attn_kvcache_evict_
from flash_attn.kvcache_interface import flash_attn_kvcache_func
