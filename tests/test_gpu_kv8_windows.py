"""Windows of flash_attn_with_quantized_kvcache with more queries than keys, where the first queries stand in front of the first
key: a negative side has no end, and a side as long as the capacity is as long as it says."""
import pytest
import torch

from kv8_util import Cache
from test_gpu_kv8_attention import _check, _q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [(18, -1), (0, -1), (-1, 70), (-1, 150), (18, 150), (200, -1), (200, 300)])
@pytest.mark.parametrize("alibi", [False, True])
#     few rows, rows over the codes, rows over the cache read back, and above head dim 128
@pytest.mark.parametrize("b,sq,h,hk,d,lens", [(2, 60, 1, 1, 80, [40, 3]), (2, 100, 3, 1, 80, [60, 90]), (2, 300, 8, 2, 128, [90, 64]),
                                              (2, 200, 4, 2, 256, [90, 150])])
def test_more_queries_than_keys(b, sq, h, hk, d, lens, alibi, window):
    cache = Cache(b, max(lens), hk, d, 16, 32, seed=250)
    slopes = torch.rand(b, h, generator=torch.Generator().manual_seed(251)) * 0.3 if alibi else None
    _check(cache, lens, _q((b, sq, h, d), "bf16", 252), "bf16", window=window, slopes=slopes)


@pytest.mark.parametrize("counts", [[300, 2], [70, 300]])
def test_ragged(counts):
    cache = Cache(2, 90, 2, 128, 16, 32, seed=253)
    _check(cache, [90, 64], _q((sum(counts), 8, 128), "bf16", 254), "bf16", window=(18, -1), ragged=counts)
