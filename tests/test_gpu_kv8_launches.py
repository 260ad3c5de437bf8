"""Which kernels a call over an 8-bit KV cache launches, for few rows, rows over the codes and rows over the cache read back,
with and without parts: those built for it alone (without packed fp32 instructions), none of the 16-bit cache's."""
import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from kv8_util import Cache
from test_gpu_kv8_attention import _q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,alibi", [(64, False), (96, False), (128, True), (256, False), (256, True)])
@pytest.mark.parametrize("sq", [1, 16, 80, 600])
@pytest.mark.parametrize("num_splits", [1, 3])
def test_only_kernels_of_its_own(d, alibi, sq, num_splits):
    import vllm_flash_attn as fa
    cache = Cache(2, 2000, 2, d, 16, 16, seed=240)
    q, slopes = _q((2, sq, 4, d), "bf16", 241).cuda(), torch.rand(4).cuda() if alibi else None
    kw = dict(cache_seqlens=torch.tensor([2000, 1801], dtype=torch.int32).cuda(), block_table=cache.block_table(), causal=True,
              alibi_slopes=slopes, num_splits=num_splits)
    gpu = cache.gpu()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        fa.flash_attn_with_quantized_kvcache(q, *gpu, **kw)
        torch.cuda.synchronize()
    names = [e.name for e in prof.events() if "vfa::" in e.name]
    assert names and all("kv8" in n for n in names), names
