"""8-bit KV cache: quantize_kvcache and dequantize_kvcache against the definition in 64 bits, bit for bit (a code is one
rounding of an exact product and reading back is exact, so nothing may differ)."""
import pytest
import torch

from kv8_util import TDT, Cache, write_ref

pytestmark = pytest.mark.gpu


def _fa():
    import vllm_flash_attn as fa
    return fa


def _same(gpu, cache):
    for t, want in zip(gpu[:2], cache.codes):
        got = t.view(torch.uint8).cpu().to(torch.int32)
        nan = (want & 127) == 127
        assert torch.equal(nan, (got & 127) == 127)
        assert torch.equal(got[~nan], want[~nan])
    for t, want in zip(gpu[2:], cache.scales):
        assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)


def _tokens(n, hk, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hk, d, generator=g) * torch.exp(spread * torch.randn(n, hk, 1, generator=g))
    return x.to(TDT[dtype])


#       b, cap, hk,  d, blk, page, starts,        news
CASES = [
    (1, 64, 1, 16, 16, 0, [0], [1]),
    (1, 64, 1, 16, 16, 16, [0], [64]),
    (3, 200, 2, 64, 16, 0, [0, 15, 16], [17, 1, 16]),
    (3, 200, 2, 64, 16, 16, [0, 15, 31], [17, 1, 2]),
    (4, 300, 8, 128, 32, 64, [0, 31, 64, 250], [300, 2, 1, 49]),
    (2, 500, 3, 80, 48, 48, [1, 47], [200, 97]),
    (2, 400, 5, 96, 64, 192, [63, 130], [66, 129]),
    (2, 300, 2, 256, 128, 128, [5, 127], [250, 1]),
    (2, 300, 1, 240, 32, 96, [95, 96], [33, 32]),
    (5, 64, 4, 112, 16, 32, [0, 3, 63, 10, 64], [0, 5, 1, 0, 3]),     # none; the last goes past the capacity
    (1, 1100, 16, 64, 512, 0, [500], [600]),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,cap,hk,d,blk,page,starts,news", CASES)
def test_ragged_write_matches_the_definition(b, cap, hk, d, blk, page, starts, news, dtype):
    cache = Cache(b, cap, hk, d, blk, page, seed=1)
    gpu = cache.gpu()
    k, v = _tokens(sum(news), hk, d, dtype, 2), _tokens(sum(news), hk, d, dtype, 3, 2.0)
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    _fa().quantize_kvcache(k.cuda(), v.cuda(), *gpu, torch.tensor(starts, dtype=torch.int32).cuda(),
                           block_table=cache.block_table(), cu_seqlens=cu.cuda(), max_seqlen=max(news))
    for i in range(b):
        for w, x in enumerate((k, v)):
            write_ref(cache, w, i, starts[i], x[cu[i]:cu[i + 1]], dtype)
    _same(gpu, cache)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_token_by_token_grows_scales_and_reencodes(dtype):
    """Loudness rises and falls from token to token: every growth re-encodes what the block holds."""
    b, hk, d = 2, 3, 64
    cache = Cache(b, 64, hk, d, 32, 32, seed=4)
    gpu, table = cache.gpu(), cache.block_table()
    g = torch.Generator().manual_seed(5)
    for t in range(48):
        x = [(torch.randn(b, 1, hk, d, generator=g) * torch.exp2(torch.randint(-6, 7, (b, 1, hk, 1), generator=g).float())).to(TDT[dtype])
             for _ in range(2)]
        starts = [t, min(t + 3, 63)]
        _fa().quantize_kvcache(x[0].cuda(), x[1].cuda(), *gpu, torch.tensor(starts, dtype=torch.int32).cuda(), block_table=table)
        for i in range(b):
            for w in range(2):
                write_ref(cache, w, i, starts[i], x[w][i], dtype)
        if t % 8 == 7:
            _same(gpu, cache)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_special_values(dtype):
    """NaN, infinities, zeros, subnormals, the type's largest and smallest values, each head another mixture."""
    big = torch.finfo(TDT[dtype]).max
    tiny = torch.finfo(TDT[dtype]).smallest_normal
    sub = tiny * torch.finfo(TDT[dtype]).eps
    rows = [[float("nan"), 1.0, -2.0], [float("inf"), 3.0, float("-inf")], [0.0, -0.0, 0.0], [sub, -3 * sub, tiny],
            [big, 1.0, -big], [big / 2, tiny, 0.3], [big * 0.96875, 7.0, -big * 0.9375], [float("nan"), float("inf"), 0.0]]
    hk, d = len(rows), 48
    x = torch.tensor(rows).repeat(1, 16).view(1, 1, hk, d).to(TDT[dtype])
    x = torch.cat((x, x.flip(-1) * 0.3, x), 1)
    cache = Cache(1, 32, hk, d, 16, 0, seed=6)
    gpu = cache.gpu()
    # starts at 1: token 0 (a random one) is held, and re-encoded where the new ones are louder
    _fa().quantize_kvcache(x.cuda(), x.cuda(), *gpu, torch.tensor([1], dtype=torch.int32).cuda())
    for w in range(2):
        write_ref(cache, w, 0, 1, x[0], dtype)
    _same(gpu, cache)
    # a fresh block: the scale is the new tokens' own; what is read back is finite where the tokens were
    _fa().quantize_kvcache(x.cuda(), x.cuda(), *gpu, torch.tensor([16], dtype=torch.int32).cuda())
    for w in range(2):
        write_ref(cache, w, 0, 16, x[0], dtype)
    _same(gpu, cache)
    k, _ = _fa().dequantize_kvcache(*gpu, torch.tensor([19], dtype=torch.int32).cuda(), max_seqlen=19, dtype=TDT[dtype])
    assert torch.equal(torch.isfinite(k[0, 16:]).cpu(), torch.isfinite(x[0]))


def test_strided_inputs_caches_and_scales():
    """k and v slices of one packed projection, a cache with K and V of a page side by side and heads outside rows."""
    b, hk, d, page, blk, pages = 2, 4, 64, 32, 16, 9
    g = torch.Generator().manual_seed(7)
    cache = Cache(b, 128, hk, d, blk, page, extra_pages=1, seed=7)
    assert cache.codes[0].shape[0] == pages
    both = torch.empty(pages, 2, hk, page, d, dtype=torch.uint8, device="cuda")
    sboth = torch.empty(pages, hk, 2, page // blk, dtype=torch.uint8, device="cuda")
    for w in range(2):
        both[:, w] = cache.codes[w].to(torch.uint8).cuda().permute(0, 2, 1, 3)
        sboth[:, :, w] = cache.scales[w].to(torch.uint8).cuda().permute(0, 2, 1)
    kc, vc = (both[:, w].permute(0, 2, 1, 3).view(torch.float8_e4m3fn) for w in range(2))
    ks, vs = (sboth[:, :, w].permute(0, 2, 1).view(torch.float8_e8m0fnu) for w in range(2))
    packed = torch.randn(b, 37, 3 * hk * d + 8, generator=g).to(torch.bfloat16)
    k, v = (packed[..., o:o + hk * d].view(b, 37, hk, d) for o in (hk * d, 2 * hk * d))
    kg, vg = (packed.cuda()[..., o:o + hk * d].view(b, 37, hk, d) for o in (hk * d, 2 * hk * d))
    starts = [3, 64]
    _fa().quantize_kvcache(kg, vg, kc, vc, ks, vs, torch.tensor(starts, dtype=torch.int32).cuda(), block_table=cache.block_table())
    for i in range(b):
        write_ref(cache, 0, i, starts[i], k[i], "bf16")
        write_ref(cache, 1, i, starts[i], v[i], "bf16")
    _same((kc, vc, ks, vs), cache)
    # inputs whose rows are not 16-byte aligned are taken too
    odd = torch.randn(b * 5 * hk * d + 1, generator=g).to(torch.bfloat16).cuda()[1:].view(b, 5, hk, d)
    _fa().quantize_kvcache(odd, odd, kc, vc, ks, vs, torch.tensor([40, 101], dtype=torch.int32).cuda(), block_table=cache.block_table())
    for i in range(b):
        for w in range(2):
            write_ref(cache, w, i, [40, 101][i], odd[i].cpu(), "bf16")
    _same((kc, vc, ks, vs), cache)


def test_cache_batch_idx_int_length_and_pages_outside_the_pool():
    hk, d = 2, 32
    cache = Cache(4, 64, hk, d, 16, 0, seed=8, batch_rows=6)
    gpu = cache.gpu()
    idx = torch.tensor([5, 0, 9, -1], dtype=torch.int32)       # the last two name no row of the cache: nothing is written
    x = _tokens(4 * 3, hk, d, "fp16", 9).view(4, 3, hk, d)
    _fa().quantize_kvcache(x.cuda(), x.cuda(), *gpu, 7, cache_batch_idx=idx.cuda())
    for i in range(2):
        for w in range(2):
            write_ref(cache, w, i, 7, x[i], "fp16", rows_of=idx)
    _same(gpu, cache)
    k, v = _fa().dequantize_kvcache(*gpu, torch.tensor([10, 3, 4, 5], dtype=torch.int32).cuda(), max_seqlen=12,
                                    cache_batch_idx=idx.cuda(), dtype=torch.float16)
    for i, n in ((0, 10), (1, 3)):
        assert torch.equal(k[i, :n].cpu().double(), cache.values(0, i, n, rows_of=idx))
        assert torch.equal(v[i, :n].cpu().double(), cache.values(1, i, n, rows_of=idx))
        assert not k[i, n:].any() and not v[i, n:].any()
    for i, n in ((2, 4), (3, 5)):
        assert torch.isnan(k[i, :n]).all() and torch.isnan(v[i, :n]).all() and not k[i, n:].any()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,cap,hk,d,blk,page,lens", [
    (1, 16, 1, 16, 16, 0, [1]),
    (3, 200, 2, 64, 16, 16, [200, 0, 33]),
    (3, 200, 3, 80, 16, 0, [7, 192, 100]),
    (4, 500, 8, 128, 32, 64, [500, 1, 64, 65]),
    (2, 300, 2, 256, 64, 192, [193, 300]),
    (2, 100, 1, 240, 48, 48, [49, 95]),
])
def test_read_back_padded_and_ragged(b, cap, hk, d, blk, page, lens, dtype):
    cache = Cache(b, cap, hk, d, blk, page, seed=10)
    gpu, table = cache.gpu(), cache.block_table()
    gl = torch.tensor(lens, dtype=torch.int32).cuda()
    want = [[cache.values(w, i, n) for i, n in enumerate(lens)] for w in range(2)]
    for most in (max(lens), max(lens) + 5, max(1, max(lens) // 2)):
        got = _fa().dequantize_kvcache(*gpu, gl, max_seqlen=most, block_table=table, dtype=TDT[dtype])
        for w in range(2):
            assert got[w].shape == (b, most, hk, d) and got[w].dtype == TDT[dtype]
            for i, n in enumerate(lens):
                n = min(n, most)
                assert torch.equal(got[w][i, :n].cpu().double(), want[w][i][:n])
                assert not got[w][i, n:].any()
    # ragged, with a gap behind the second sequence and rows behind the last one
    room = [n + (4 if i == 1 else 0) for i, n in enumerate(lens)]
    cu = torch.tensor([0] + room).cumsum(0).to(torch.int32)
    total = int(cu[-1]) + 3
    got = _fa().dequantize_kvcache(*gpu, gl, cu_seqlens=cu.cuda(), total_seqlen=total, block_table=table, dtype=TDT[dtype])
    for w in range(2):
        assert got[w].shape == (total, hk, d)
        full = torch.zeros(total, hk, d, dtype=torch.float64)
        for i, n in enumerate(lens):
            full[cu[i]:cu[i] + n] = want[w][i]
        assert torch.equal(got[w].cpu().double(), full)


def test_offsets_past_32_bits():
    """The last pages of a pool of more than 2^32 bytes are written and read."""
    pages, page, hk, d, blk = 4200, 512, 16, 128, 64
    kc = torch.zeros(pages, page, hk, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ks = torch.zeros(pages, page // blk, hk, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    assert kc.numel() > 2 ** 32
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(1, 1100, hk, d, device="cuda", generator=g).to(torch.bfloat16)
    _fa().quantize_kvcache(x, x, kc, kc.clone(), ks, ks.clone(), torch.tensor([100], dtype=torch.int32, device="cuda"), block_table=table)
    k, _ = _fa().dequantize_kvcache(kc, kc, ks, ks, torch.tensor([1200], dtype=torch.int32, device="cuda"), max_seqlen=1200, block_table=table)
    # e4m3: half a step of 2^-4 of the value, or of the smallest step 2^-9 under a scale of at most max / 224
    err = (k[0, 100:].float() - x[0].float()).abs()
    assert bool((err <= x[0].float().abs() * 2.0 ** -4 + x.abs().max().float() / 224 * 2.0 ** -10).all())
    assert not k[0, :100].any()
    assert not kc[1:pages - 2].view(torch.uint8).any()
