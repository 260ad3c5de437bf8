"""Attention over an 8-bit KV cache at the longest capacity there can be, 2^30 tokens: positions, windows and their sums."""
import pytest
import torch

from kv8_util import Cache, attend_ref
from test_gpu_kv8_attention import _close, _q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sq", [1, 3, 100])
@pytest.mark.parametrize("lens", [2 ** 30, 2 ** 30 - 5])
@pytest.mark.parametrize("causal,window", [(False, (50, -1)), (True, (50, -1)), (False, (50, 2 ** 30 - 1)), (False, (50, 7))])
def test_a_full_sequence_of_the_longest_capacity(causal, window, lens, sq):
    import vllm_flash_attn as fa
    page, d = 16384, 16
    cache = Cache(1, page, 1, d, page, page, extra_pages=0, seed=210)      # one page, at every place of the table
    table = torch.zeros(1, 2 ** 30 // page, dtype=torch.int32).cuda()
    q = _q((1, sq, 1, d), "bf16", 211).cuda()
    out = fa.flash_attn_with_quantized_kvcache(q, *cache.gpu(), cache_seqlens=torch.tensor([lens], dtype=torch.int32).cuda(),
                                               block_table=table, causal=causal, window_size=window)
    n = page - (2 ** 30 - lens)                        # (the last page alone: the window lies in it)
    assert n > sq + 50
    want, tol = attend_ref(q[0], cache.values(0, 0, n), cache.values(1, 0, n), causal, window)
    _close(out[0], want, tol)


def test_appending_as_many_tokens_to_a_full_sequence():
    """2^30 cached and 2^30 new tokens: the new ones are dropped, the old ones attended."""
    import vllm_flash_attn as fa
    page, d = 16384, 16
    cache = Cache(1, page, 1, d, page, page, extra_pages=0, seed=212)
    gpu = cache.gpu()
    table = torch.zeros(1, 2 ** 30 // page, dtype=torch.int32).cuda()
    q, x = _q((1, 1, 1, d), "bf16", 213).cuda(), _q((1, 1, 1, d), "bf16", 214).cuda().expand(1, 2 ** 30, 1, d)
    kw = dict(cache_seqlens=torch.tensor([2 ** 30], dtype=torch.int32).cuda(), block_table=table, window_size=(50, 0))
    before = [t.view(torch.uint8).clone() for t in gpu]
    out = fa.flash_attn_with_quantized_kvcache(q, *gpu, k=x, v=x, **kw)
    want, tol = attend_ref(q[0], cache.values(0, 0, page), cache.values(1, 0, page), True, (50, 0))
    _close(out[0], want, tol)
    for a, b in zip(before, gpu):
        assert torch.equal(a, b.view(torch.uint8))
