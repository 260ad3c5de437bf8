"""Attention over an 8-bit KV cache where what a row does not see cannot be multiplied by zero: NaN codes and scales, pages
outside the pool, values past fp16's range.  A key that no row of its sequence sees has no part in any result, and a row that
sees no key is zero."""
import pytest
import torch

from kv8_util import TDT, Cache, attend_ref
from test_gpu_kv8_attention import _close, _q

pytestmark = pytest.mark.gpu


def _fa():
    import vllm_flash_attn as fa
    return fa


def _spoil(cache, gpu, i, tokens, how, table):
    """Makes the given tokens of sequence i unusable, K and V, in the call's tensors alone: the host mirror stays clean."""
    for tok in tokens:
        page, row = cache.place(i, tok)
        if how == "page":
            table[i, tok // cache.page] = -1
        for w in range(2):
            codes, scales = gpu[w].view(torch.uint8), gpu[2 + w].view(torch.uint8)
            if how == "code":
                codes[page, row] = 127
            elif how == "scale":
                scales[page, row // cache.blk] = 255
            elif how == "large":                       # 448 * 2^20: an infinity in fp16
                codes[page, row] = 126
                scales[page, row // cache.blk] = 147


#     sq, h, hk, d, lens: few rows, rows over the codes, rows over the cache read back
SHAPES = [(2, 8, 2, 128, [300, 190]), (1, 4, 4, 64, [115, 90]), (60, 8, 2, 128, [330, 190]), (30, 4, 2, 256, [300, 190]), (80, 1, 1, 64, [355, 158]),
          (300, 8, 2, 128, [900, 640]), (1100, 1, 1, 64, [1300, 1500]), (270, 8, 2, 96, [700, 500]),
          (100, 4, 2, 256, [500, 333]), (200, 2, 2, 160, [500, 333]), (270, 8, 2, 128, [3000, 2011])]


@pytest.mark.parametrize("how", ["page", "code", "scale", "large"])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("sq,h,hk,d,lens", SHAPES)
def test_keys_in_front_of_the_window(sq, h, hk, d, lens, ragged, how):
    dtype = "fp16" if how == "large" else "bf16"
    wl = 40
    cache = Cache(2, max(lens), hk, d, 16, 32, seed=200)
    gpu, table = cache.gpu(), cache.block_table()
    counts = [sq, 1] if ragged else [sq, sq]
    for i, n in enumerate(lens):
        first = n - counts[i] - wl                     # the first key that a row sees
        unit = 32 if how == "page" else 16 if how in ("scale", "large") else 1
        _spoil(cache, gpu, i, range(0, first // unit * unit), how, table)
    q = _q((sum(counts), h, d) if ragged else (2, sq, h, d), dtype, 201)
    kw = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=table, window_size=(wl, 0))
    if ragged:
        kw.update(cu_seqlens_q=torch.tensor([0, sq, sq + 1], dtype=torch.int32).cuda(), max_seqlen_q=sq)
    out = _fa().flash_attn_with_quantized_kvcache(q.cuda(), *gpu, **kw)
    for i, n in enumerate(lens):
        qi, oi = (q[i], out[i]) if not ragged else (q[:sq], out[:sq]) if i == 0 else (q[sq:], out[sq:])
        want, tol = attend_ref(qi.cuda(), cache.values(0, i, n), cache.values(1, i, n), True, (wl, 0), dtype=dtype)
        _close(oi, want, tol, "sequence %d" % i)


#     sq, h, hk, d, lens: more query positions than keys
SHORT = [(12, 4, 2, 64, [5, 9]), (7, 4, 4, 64, [3, 6]), (16, 8, 2, 128, [9, 2]), (9, 4, 2, 256, [5, 8]),
         (50, 8, 2, 128, [33, 49]), (150, 2, 2, 64, [20, 149]), (40, 4, 2, 256, [17, 39]),
         (300, 8, 2, 128, [40, 299]), (1100, 1, 1, 64, [50, 1000]), (270, 8, 2, 96, [100, 3]), (100, 4, 2, 256, [33, 95]), (200, 2, 2, 160, [7, 180])]


@pytest.mark.parametrize("how", ["page", "code", "large"])
@pytest.mark.parametrize("num_splits", [1, 3])
@pytest.mark.parametrize("sq,h,hk,d,lens", SHORT)
def test_a_row_that_sees_no_key_is_zero(sq, h, hk, d, lens, num_splits, how):
    dtype = "fp16" if how == "large" else "bf16"
    cache = Cache(2, max(lens), hk, d, 16, 16, seed=202)
    gpu, table = cache.gpu(), cache.block_table()
    for i, n in enumerate(lens):
        _spoil(cache, gpu, i, [n - 1], how, table)     # a key that the last row sees
    q = _q((2, sq, h, d), dtype, 203).cuda()
    lens_gpu = torch.tensor(lens, dtype=torch.int32).cuda()
    out = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=lens_gpu, block_table=table, causal=True, num_splits=num_splits)
    for i, n in enumerate(lens):
        assert not out[i, :sq - n].any(), "sequence %d: rows that see no key are not zero" % i
        if how != "large":
            assert torch.isnan(out[i, sq - 1]).all()
    assert out.dtype == TDT[dtype]
