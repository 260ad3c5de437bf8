"""flash_attn_with_quantized_kvcache against attention in 64 bits over the values that the cache stands for; tolerances
from the number formats (attend_ref)."""
import pytest
import torch

from kv8_util import TDT, Cache, attend_ref, write_ref

pytestmark = pytest.mark.gpu


def _fa():
    import vllm_flash_attn as fa
    return fa


def _q(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TDT[dtype])


def _close(got, want, tol, what=""):
    got = got.double().to(want.device)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g over %.3g" % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].nan_to_num(9e9).max()), float(tol[bad].min()))


def _check(cache, lens, q, dtype, rows_of=None, ragged=None, news=None, **kw):
    """q dense (b, sq, h, d) or ragged with `ragged` query counts; `news`: new k, v."""
    fa, gpu = _fa(), cache.gpu()
    args = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=cache.block_table(),
                causal=kw.get("causal", False), window_size=kw.get("window", (-1, -1)), num_splits=kw.get("num_splits", 0),
                softmax_scale=kw.get("scale"))
    slopes = kw.get("slopes")
    if slopes is not None:
        args["alibi_slopes"] = slopes.cuda()
    if rows_of is not None:
        args["cache_batch_idx"] = rows_of.cuda()
    if ragged is not None:
        cu = torch.tensor([0] + ragged).cumsum(0).to(torch.int32)
        args.update(cu_seqlens_q=cu.cuda(), max_seqlen_q=max(ragged))
    total = list(lens)
    if news is not None:
        args.update(k=news[0].cuda(), v=news[1].cuda())
        for i in range(cache.b):
            for w in range(2):
                write_ref(cache, w, i, lens[i], news[w][i], dtype, rows_of)
        total = [min(n + news[0].shape[1], cache.cap) for n in lens]
    out = fa.flash_attn_with_quantized_kvcache(q.cuda(), *gpu, **args)
    assert out.shape == q.shape and out.dtype == q.dtype
    for i, n in enumerate(total):
        qi = q[i] if ragged is None else q[cu[i]:cu[i + 1]]
        oi = out[i] if ragged is None else out[cu[i]:cu[i + 1]]
        if qi.shape[0] == 0:
            continue
        sl = None if slopes is None else (slopes if slopes.dim() == 1 else slopes[i])
        want, tol = attend_ref(qi.cuda(), cache.values(0, i, n, rows_of), cache.values(1, i, n, rows_of),
                               args["causal"], args["window_size"], sl, args["softmax_scale"], dtype)
        _close(oi, want, tol, "sequence %d" % i)
    return out, gpu


#       b, sq, h, hk,  d, blk, page, lens
DECODE = [
    (1, 1, 1, 1, 16, 16, 0, [1]),
    (1, 1, 4, 1, 64, 16, 16, [17]),
    (2, 1, 8, 8, 64, 16, 16, [33, 1000]),
    (3, 1, 8, 2, 128, 32, 64, [0, 31, 777]),
    (2, 1, 32, 8, 128, 64, 0, [1024, 63]),
    (2, 1, 6, 3, 80, 48, 48, [49, 301]),
    (2, 1, 7, 1, 96, 16, 32, [500, 2]),
    (2, 1, 4, 2, 256, 32, 96, [95, 333]),
    (2, 1, 16, 1, 192, 16, 16, [129, 128]),
    (2, 1, 20, 1, 128, 16, 0, [200, 100]),          # more than 16 rows a KV head
    (1, 1, 48, 1, 64, 16, 16, [700]),               # more than 32
    (5, 1, 10, 5, 240, 16, 48, [1, 15, 16, 47, 48]),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,sq,h,hk,d,blk,page,lens", DECODE)
@pytest.mark.parametrize("num_splits", [0, 1, 3])
def test_one_query_token(b, sq, h, hk, d, blk, page, lens, num_splits, dtype):
    cache = Cache(b, max(lens) + 5, hk, d, blk, page, seed=1)
    _check(cache, lens, _q((b, sq, h, d), dtype, 2), dtype, num_splits=num_splits)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal,window,alibi", [(False, (-1, -1), False), (True, (-1, -1), False), (True, (37, -1), False),
                                                 (False, (20, 10), False), (False, (-1, 3), False), (True, (-1, -1), True),
                                                 (False, (64, 0), True)])
@pytest.mark.parametrize("b,sq,h,hk,d,blk,page,lens,num_splits", [
    (2, 5, 8, 2, 128, 32, 64, [200, 77], 0),
    (2, 3, 4, 4, 64, 16, 16, [3, 300], 2),
    (3, 17, 4, 1, 96, 16, 0, [17, 100, 5], 1),       # fewer keys than queries: rows that see none
    (1, 70, 6, 2, 256, 64, 64, [500], 4),
    (2, 33, 2, 2, 80, 16, 16, [0, 40], 1),           # an empty sequence
    (1, 150, 8, 2, 128, 16, 32, [411], 0),
])
def test_masks(b, sq, h, hk, d, blk, page, lens, num_splits, causal, window, alibi, dtype):
    cache = Cache(b, max(lens) + 40, hk, d, blk, page, seed=3)
    slopes = torch.rand(b, h, generator=torch.Generator().manual_seed(4)) * 0.3 if alibi else None
    _check(cache, lens, _q((b, sq, h, d), dtype, 5), dtype, causal=causal, window=window, slopes=slopes, num_splits=num_splits)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("h,hk,d,page,counts,lens", [
    (8, 2, 128, 64, [1, 200, 1, 0, 37], [300, 210, 1, 50, 37]),
    (4, 4, 64, 16, [3, 1, 129], [3, 700, 400]),
    (2, 1, 256, 32, [65, 1], [65, 222]),
])
def test_ragged_queries(h, hk, d, page, counts, lens, dtype):
    cache = Cache(len(lens), max(lens), hk, d, 16, page, seed=6)
    _check(cache, lens, _q((sum(counts), h, d), dtype, 7), dtype, ragged=counts, causal=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,new,sq,h,hk,d,blk,page,lens", [
    (3, 1, 1, 8, 2, 128, 16, 16, [0, 15, 200]),
    (2, 4, 4, 4, 4, 64, 32, 64, [61, 62]),
    (2, 40, 7, 6, 1, 96, 16, 0, [3, 130]),
    (1, 2, 2, 2, 2, 256, 128, 128, [127]),
])
def test_append_then_attend(b, new, sq, h, hk, d, blk, page, lens, dtype):
    cache = Cache(b, max(lens) + new, hk, d, blk, page, seed=8)
    news = [_q((b, new, hk, d), dtype, 9 + w) for w in range(2)]
    _, gpu = _check(cache, lens, _q((b, sq, h, d), dtype, 11), dtype, causal=True, news=news)
    for t, want in zip(gpu[:2], cache.codes):
        assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)
    for t, want in zip(gpu[2:], cache.scales):
        assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)


def test_cache_batch_idx_scale_and_out():
    rows_of = torch.tensor([4, 0, 2], dtype=torch.int32)
    cache = Cache(3, 100, 2, 64, 16, 0, seed=12, batch_rows=5)
    q = _q((3, 2, 4, 64), "bf16", 13)
    out, gpu = _check(cache, [100, 64, 9], q, "bf16", rows_of=rows_of, causal=True, scale=0.3)
    lens = torch.tensor([100, 64, 9], dtype=torch.int32).cuda()
    kw = dict(cache_seqlens=lens, cache_batch_idx=rows_of.cuda(), causal=True, softmax_scale=0.3)
    wide = torch.empty(3, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    r = _fa().flash_attn_with_quantized_kvcache(q.cuda(), *gpu, out=wide[:, :, ::2], **kw)
    assert r.data_ptr() == wide.data_ptr() and torch.equal(wide[:, :, ::2], out)
    odd = torch.empty(3 * 2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 2, 4, 64)     # not 16-byte aligned
    r = _fa().flash_attn_with_quantized_kvcache(q.cuda(), *gpu, out=odd, **kw)
    assert r.data_ptr() == odd.data_ptr() and torch.equal(odd, out)
    qs = torch.empty(3, 2, 4, 72, dtype=torch.bfloat16, device="cuda")[..., :64]
    qs.copy_(q)
    assert torch.equal(_fa().flash_attn_with_quantized_kvcache(qs, *gpu, **kw), out)


@pytest.mark.parametrize("num_splits", [1, 4])
def test_nan_behind_the_sequence_does_not_matter_and_inside_does(num_splits):
    for d, page in ((64, 16), (128, 32), (256, 64)):
        cache = Cache(2, 200, 2, d, 16, page, seed=14)
        lens = [50, 161]
        for w in range(2):
            for i, n in enumerate(lens):
                for tok in range(n, -(-n // page) * page):
                    pg, row = cache.place(i, tok)
                    cache.codes[w][pg, row] = 127                # NaN behind the last token, to the page's end
        q = _q((2, 1, 4, d), "bf16", 15)
        _check(cache, lens, q, "bf16", num_splits=num_splits)
        # a NaN before the window's first key: no row sees it
        pg, row = cache.place(1, 3)
        cache.codes[1][pg, row] = 127
        cache.codes[0][pg, row] = 127
        _check(cache, lens, q, "bf16", num_splits=num_splits, window=(30, -1))
        out = _fa().flash_attn_with_quantized_kvcache(q.cuda(), *cache.gpu(), cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(),
                                                      block_table=cache.block_table(), num_splits=num_splits)
        assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any()


def test_a_page_outside_the_pool_gives_nan_for_its_sequence_alone():
    cache = Cache(3, 128, 2, 128, 32, 32, seed=16)
    q = _q((3, 1, 8, 128), "fp16", 17).cuda()
    gpu, table = cache.gpu(), cache.block_table()
    lens = torch.tensor([100, 128, 20], dtype=torch.int32).cuda()
    good = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=lens, block_table=table)
    for bad in (-1, 10 ** 6, cache.codes[0].shape[0]):
        t = table.clone()
        t[1, 2] = bad
        t[2, 1] = bad           # behind the third sequence's last token: never looked at
        out = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=lens, block_table=t)
        assert torch.isnan(out[1]).all()
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


def test_lengths_past_the_capacity_are_cut():
    cache = Cache(2, 64, 1, 64, 16, 16, seed=18)
    q = _q((2, 1, 2, 64), "bf16", 19).cuda()
    gpu, table = cache.gpu(), cache.block_table()
    cut = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=torch.tensor([64, 0], dtype=torch.int32).cuda(), block_table=table)
    out = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32).cuda(), block_table=table)
    assert torch.equal(out, cut) and not out[1].any()
    assert torch.equal(_fa().flash_attn_with_quantized_kvcache(q, *gpu, block_table=table)[0], cut[0])     # no lengths: all of the capacity


def test_equals_the_16_bit_path_on_the_cache_read_back():
    """The same exact values through flash_attn_with_kvcache: two kernels' roundings of P and of the result apart."""
    fa = _fa()
    for dtype in ("fp16", "bf16"):
        cache = Cache(3, 900, 4, 128, 64, 64, seed=20)
        gpu, table = cache.gpu(), cache.block_table()
        lens = [900, 411, 64]
        gl = torch.tensor(lens, dtype=torch.int32).cuda()
        q = _q((3, 2, 16, 128), dtype, 21)
        a = fa.flash_attn_with_quantized_kvcache(q.cuda(), *gpu, cache_seqlens=gl, block_table=table, causal=True)
        k, v = fa.dequantize_kvcache(*gpu, gl, max_seqlen=900, block_table=table, dtype=TDT[dtype])
        b = fa.flash_attn_with_kvcache(q.cuda(), k, v, cache_seqlens=gl, causal=True)
        for i, n in enumerate(lens):
            _, tol = attend_ref(q[i].cuda(), cache.values(0, i, n), cache.values(1, i, n), True, dtype=dtype)
            assert bool(((a[i].double() - b[i].double()).abs() <= 2 * tol).all())


def test_repeated_calls_give_the_same_bits():
    cache = Cache(4, 3000, 2, 128, 64, 64, seed=22)
    gpu, table = cache.gpu(), cache.block_table()
    q = _q((4, 1, 8, 128), "bf16", 23).cuda()
    lens = torch.tensor([3000, 5, 1999, 640], dtype=torch.int32).cuda()
    first = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=lens, block_table=table)
    for _ in range(20):
        assert torch.equal(first, _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=lens, block_table=table))
