"""The caller's `out` of flash_attn_with_quantized_kvcache: rows behind the last sequence stay as they were, whatever its
alignment, and what is returned is the caller's tensor also where there is nothing to compute."""
import pytest
import torch

from kv8_util import Cache
from test_gpu_kv8_attention import _q

pytestmark = pytest.mark.gpu


def _outs(shape):
    n = 1
    for x in shape:
        n *= x
    yield torch.full(shape, 7.0, dtype=torch.bfloat16, device="cuda")
    yield torch.full((n + 1,), 7.0, dtype=torch.bfloat16, device="cuda")[1:].view(shape)                  # not 16-byte aligned
    yield torch.full((*shape[:-1], shape[-1] + 4), 7.0, dtype=torch.bfloat16, device="cuda")[..., :-4]    # strides of 8 bytes


@pytest.mark.parametrize("counts", [[1, 3], [300, 2]])
def test_rows_behind_the_last_sequence_stay(counts):
    import vllm_flash_attn as fa
    cache = Cache(2, 400, 2, 128, 16, 16, seed=220)
    gpu, table = cache.gpu(), cache.block_table()
    total = sum(counts)
    q = _q((total + 5, 8, 128), "bf16", 221).cuda()
    kw = dict(cache_seqlens=torch.tensor([400, 99], dtype=torch.int32).cuda(), block_table=table, causal=True, max_seqlen_q=max(counts),
              cu_seqlens_q=torch.tensor([0, counts[0], total], dtype=torch.int32).cuda())
    want = fa.flash_attn_with_quantized_kvcache(q, *gpu, **kw)
    for out in _outs(tuple(q.shape)):
        r = fa.flash_attn_with_quantized_kvcache(q, *gpu, out=out, **kw)
        assert r.data_ptr() == out.data_ptr()
        assert torch.equal(out[:total], want[:total])
        assert bool((out[total:] == 7).all())


def test_nothing_to_compute_returns_the_callers_tensor():
    import vllm_flash_attn as fa
    cache = Cache(2, 64, 2, 64, 16, 16, seed=222)
    q = _q((5, 4, 64), "bf16", 223).cuda()
    kw = dict(cache_seqlens=torch.tensor([64, 9], dtype=torch.int32).cuda(), block_table=cache.block_table(), max_seqlen_q=0,
              cu_seqlens_q=torch.zeros(3, dtype=torch.int32).cuda())
    for out in _outs(tuple(q.shape)):
        r = fa.flash_attn_with_quantized_kvcache(q, *cache.gpu(), out=out, **kw)
        assert r.data_ptr() == out.data_ptr() and r.stride() == out.stride()
        assert bool((out == 7).all())
