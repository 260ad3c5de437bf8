"""MI355X-native drop-in for the `vllm_flash_attn` package (same names and signatures as
/root/reference/vllm_flash_attn/__init__.py:1-11), with operators beyond it: a KV cache held in 8 bits
(quantized_kvcache.py) and the norm and rotation of query and key heads in one pass (qk_norm.py)."""
__version__ = "2.5.8.post3"

from vllm_flash_attn.flash_attn_interface import (  # noqa: F401
    enable_cpu_fp32,
    flash_attn_func,
    flash_attn_kvpacked_func,
    flash_attn_qkvpacked_func,
    flash_attn_varlen_func,
    flash_attn_varlen_kvpacked_func,
    flash_attn_varlen_qkvpacked_func,
    flash_attn_with_kvcache,
)
from vllm_flash_attn.quantized_kvcache import (  # noqa: F401
    dequantize_kvcache,
    flash_attn_with_quantized_kvcache,
    quantize_kvcache,
)
from vllm_flash_attn.qk_norm import qk_norm_rotary_func  # noqa: F401
