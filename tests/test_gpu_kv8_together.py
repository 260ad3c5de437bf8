"""The operators around an 8-bit KV cache as they are used together (prompt, decode steps, read-back, training step), in
graphs, on other streams, over large pools and on the paths that only long queries or large batches take."""
import pytest
import torch

from kv8_util import HALF_STEP, TDT, Cache, attend_ref, encode, norm_rotary_ref, write_ref
from test_gpu_kv8_attention import _check, _close, _q
from test_gpu_qk_norm import test_forward_and_gradients as _norm_test

pytestmark = pytest.mark.gpu


def _fa():
    import vllm_flash_attn as fa
    return fa


def _tables(rows, rd):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    return a.cos().float(), a.sin().float()


def _normed(x, w, cos, sin, pos, dtype):
    """The formula in 64 bits and the bound of test_gpu_qk_norm.py on fp32 arithmetic with one rounding."""
    d = x.shape[-1]
    y = norm_rotary_ref(x.double(), w.double(), cos.double()[pos], sin.double()[pos], pos, 1e-6, True)
    r = 1 / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    pair = (x.double() * r * w.double()).abs().amax(-1, keepdim=True) * 2
    return y, HALF_STEP[dtype] * y.abs() + (d + 12) * 2.0 ** -24 * pair + (2.0 ** -25 if dtype == "fp16" else 0.0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("h,hk,d,blk,page", [(8, 2, 128, 16, 64), (4, 4, 64, 32, 32), (6, 1, 80, 16, 0)])
def test_prompts_decode_steps_and_read_back(h, hk, d, blk, page, dtype):
    """Ragged prompts into the cache and attended, decode steps of one or more drafted tokens, then the cache read back
    for the 16-bit kernels; after every call the cache is checked byte for byte and the output element by element."""
    fa, dt = _fa(), TDT[dtype]
    prompts, steps, rd = [37, 1, 90], [1, 3, 1, 1, 16], d // 32 * 32
    b, cap = len(prompts), max(prompts) + sum(steps)
    cache = Cache(b, cap, hk, d, blk, page, seed=30)
    gpu, table = cache.gpu(), cache.block_table()
    cos, sin = _tables(cap, rd)
    gc, gs = cos.cuda(), sin.cuda()
    w = [(1 + 0.2 * torch.randn(d, generator=torch.Generator().manual_seed(31 + i))).to(dt) for i in range(2)]
    gw = [x.cuda() for x in w]
    lens = [0] * b

    def tokens(n, seed):                 # packed projections: q, k and v side by side
        x = _q((n, (h + 2 * hk) * d), dtype, seed)
        return x, x.cuda()

    def split(x):
        a = x.unflatten(-1, (h + 2 * hk, d))
        return a[..., :h, :], a[..., h:h + hk, :], a[..., h + hk:, :]

    def same_cache():
        for t, want in zip(gpu[:2], cache.codes):
            assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)
        for t, want in zip(gpu[2:], cache.scales):
            assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)

    # prompts: one ragged batch
    x, gx = tokens(sum(prompts), 33)
    pos = torch.cat([torch.arange(n) for n in prompts])
    cu = torch.tensor([0] + prompts).cumsum(0).to(torch.int32)
    q, k, v = split(gx)
    q2, k2 = fa.qk_norm_rotary_func(q, k, *gw, gc, gs, positions=pos.to(torch.int32).cuda())
    for got, src, i in ((q2, split(x)[0], 0), (k2, split(x)[1], 1)):
        want, tol = _normed(src[None], w[i], cos, sin, pos[None], dtype)
        _close(got[None], want, tol, "prompt norm")
    zero = torch.zeros(b, dtype=torch.int32).cuda()
    fa.quantize_kvcache(k2, v, *gpu, zero, block_table=table, cu_seqlens=cu.cuda(), max_seqlen=max(prompts))
    for i in range(b):
        write_ref(cache, 0, i, 0, k2[cu[i]:cu[i + 1]].cpu(), dtype)
        write_ref(cache, 1, i, 0, split(x)[2][cu[i]:cu[i + 1]], dtype)
    lens = list(prompts)
    same_cache()
    out = fa.flash_attn_with_quantized_kvcache(q2, *gpu, cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=table,
                                               cu_seqlens_q=cu.cuda(), max_seqlen_q=max(prompts), causal=True)
    for i, n in enumerate(lens):
        want, tol = attend_ref(q2[cu[i]:cu[i + 1]], cache.values(0, i, n), cache.values(1, i, n), True, dtype=dtype)
        _close(out[cu[i]:cu[i + 1]], want, tol, "prompt %d" % i)

    for s, n_new in enumerate(steps):
        x, gx = tokens(b * n_new, 40 + s)
        pos = torch.tensor(lens)[:, None] + torch.arange(n_new)
        q, k, v = (t.unflatten(0, (b, n_new)) for t in split(gx))
        q2, k2 = fa.qk_norm_rotary_func(q, k, *gw, gc, gs, positions=pos.to(torch.int32).cuda())
        want, tol = _normed(split(x)[0].unflatten(0, (b, n_new)), w[0], cos, sin, pos, dtype)
        _close(q2, want, tol, "step norm")
        out = fa.flash_attn_with_quantized_kvcache(q2, *gpu, k=k2, v=v, cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(),
                                                   block_table=table, causal=True)
        for i in range(b):
            write_ref(cache, 0, i, lens[i], k2[i].cpu(), dtype)
            write_ref(cache, 1, i, lens[i], v[i].cpu(), dtype)
            lens[i] += n_new
        same_cache()
        for i, n in enumerate(lens):
            want, tol = attend_ref(q2[i], cache.values(0, i, n), cache.values(1, i, n), True, dtype=dtype)
            _close(out[i], want, tol, "step %d sequence %d" % (s, i))

    cu_k = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    k16, v16 = fa.dequantize_kvcache(*gpu, torch.tensor(lens, dtype=torch.int32).cuda(), cu_seqlens=cu_k.cuda(), total_seqlen=int(cu_k[-1]),
                                     block_table=table, dtype=dt)
    n_new = steps[-1]
    cu_q = torch.arange(0, (b + 1) * n_new, n_new, dtype=torch.int32).cuda()
    again = fa.flash_attn_varlen_func(q2.flatten(0, 1), k16, v16, cu_q, cu_k.cuda(), n_new, max(lens), causal=True)
    for i, n in enumerate(lens):
        assert torch.equal(k16[cu_k[i]:cu_k[i + 1]].double().cpu(), cache.values(0, i, n))
        want, tol = attend_ref(q2[i], cache.values(0, i, n), cache.values(1, i, n), True, dtype=dtype)
        _close(again[i * n_new:(i + 1) * n_new], want, tol, "read back %d" % i)


@pytest.mark.parametrize("shape", [(3, 50, 1, 1, 128, 64, False), (2, 33, 4, 1, 64, 32, True), (1, 7, 2, 2, 128, 128, True), (5, 9, 3, 1, 40, 16, False),
                                   (2, 21, 16, 1, 256, 256, False), (70, 1, 2, 1, 64, 64, False)])
@pytest.mark.parametrize("given", [False, True])
def test_norm_of_few_heads(shape, given):
    """Tokens of so few heads that several share a wave, on one side or on both; the last ones alone."""
    b, s, h, hk, d, rd, inter = shape
    for dtype in ("fp16", "bf16"):
        _norm_test(b, s, h, hk, d, rd, inter, "fp32", "same", given, dtype)


def test_training_step_through_the_attention():
    """loss(attention(norm(q), norm(k), v)): the gradients that reach the norm's inputs are the formula's for the gradient
    that the attention hands over."""
    fa = _fa()
    g = torch.Generator().manual_seed(50)
    b, s, h, hk, d = 2, 65, 4, 2, 64
    leaves = [t.cuda().requires_grad_() for t in (*(torch.randn(b, s, n, d, generator=g).bfloat16() for n in (h, hk, hk)),
                                                  1 + 0.1 * torch.randn(d, generator=g), 1 + 0.1 * torch.randn(d, generator=g))]
    q, k, v, wq, wk = leaves
    cos, sin = (t.cuda() for t in _tables(s, d))
    q2, k2 = fa.qk_norm_rotary_func(q, k, wq, wk, cos, sin)
    out = fa.flash_attn_func(q2, k2, v, causal=True, deterministic=True)
    dout = torch.randn(out.shape, generator=g).bfloat16().cuda()
    dq2, dk2 = torch.autograd.grad(out, (q2, k2), dout, retain_graph=True)
    got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    want = torch.autograd.grad((q2, k2), (q, k, wq, wk), (dq2, dk2))
    for a, b_ in zip((got[0], got[1], got[3], got[4]), want):
        assert torch.equal(a, b_)
    u = HALF_STEP["bf16"]
    for x, w, dy, gx, gw in ((q, wq, dq2, got[0], got[3]), (k, wk, dk2, got[1], got[4])):
        xd, wd = x.detach().cpu().double().requires_grad_(), w.detach().cpu().double().requires_grad_()
        pos = torch.arange(s).expand(b, s)
        y = norm_rotary_ref(xd, wd, cos.cpu().double()[pos], sin.cpu().double()[pos], pos, 1e-6, True)
        dx, dw = torch.autograd.grad(y, (xd, wd), dy.cpu().double())
        r = 1 / (xd.detach().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        xr = (xd.detach() * r).abs()
        gmax = dy.cpu().double().abs().amax(-1, keepdim=True) * 2
        size = r * gmax * wd.detach().abs().max() * (1 + xr * xr.mean(-1, keepdim=True))
        assert bool(((gx.cpu().double() - dx).abs() <= u * dx.abs() + 2 * (d + 12) * 2.0 ** -24 * size).all())
        assert bool(((gw.cpu().double() - dw).abs() <= 2.0 ** -24 * dw.abs() + (b * s * x.shape[2] + d + 12) * 2.0 ** -24 * (gmax * xr).sum((0, 1, 2))).all())


def _decode_state(seed, b=3, h=8, hk=2, d=128):
    cache = Cache(b, 3000, hk, d, 16, 64, seed=seed)
    g = torch.Generator().manual_seed(seed)
    s = dict(x=torch.randn(b, 1, (h + 2 * hk) * d, generator=g).bfloat16().cuda(), lens=torch.tensor([2000, 5, 640], dtype=torch.int32).cuda(),
             w=torch.ones(d).bfloat16().cuda(), gpu=cache.gpu(), table=cache.block_table())
    s["cos"], s["sin"] = (t.cuda() for t in _tables(3000, d))
    return s


def _decode_step(s, h=8, hk=2, d=128):
    fa = _fa()
    a = s["x"].unflatten(-1, (h + 2 * hk, d))
    q, k = fa.qk_norm_rotary_func(a[..., :h, :], a[..., h:h + hk, :], s["w"], s["w"], s["cos"], s["sin"], positions=s["lens"][:, None])
    return fa.flash_attn_with_quantized_kvcache(q, *s["gpu"], k=k, v=a[..., h + hk:, :], cache_seqlens=s["lens"], block_table=s["table"], causal=True)


def _copy(s):
    return {n: tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone() for n, x in s.items()}


def _bytes(s):
    return [t.view(torch.uint8) for t in s["gpu"]]


def test_two_captured_decode_steps_replayed_in_turn():
    """Norm, append, attention split over the keys and its merge, as two graphs of two states that share nothing but the
    allocator's pool; each replay (with new tokens, longer sequences and eager calls between) against the eager step."""
    states = [_decode_state(60), _decode_state(61)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            _decode_step(_copy(s))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(_decode_step(s))
        graphs.append(g)
    gen = torch.Generator().manual_seed(62)
    for turn in range(5):
        eager = []
        for s in states:
            s["x"].copy_(torch.randn(s["x"].shape, generator=gen).bfloat16())
            s["lens"].add_(turn)
            c = _copy(s)
            eager.append((_decode_step(c), c))
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager[i][0]), (turn, i)
            for a, b in zip(_bytes(states[i]), _bytes(eager[i][1])):
                assert torch.equal(a, b)


def test_captured_write_and_read_back():
    cache = Cache(2, 200, 2, 64, 16, 32, seed=63)
    gpu, table = cache.gpu(), cache.block_table()
    lens = torch.tensor([0, 30], dtype=torch.int32).cuda()
    k, v = (_q((2, 50, 2, 64), "fp16", 64 + i).cuda() for i in range(2))

    def call(gpu, lens):
        _fa().quantize_kvcache(k, v, *gpu, lens, block_table=table)
        return _fa().dequantize_kvcache(*gpu, lens + 50, max_seqlen=160, block_table=table, dtype=torch.float16)

    call([t.clone() for t in gpu], lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(gpu, lens)
    for turn in range(4):
        k.mul_(1.5)
        lens.add_(7)
        mine = [t.clone() for t in gpu]
        want = call(mine, lens)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*out, *(t.view(torch.uint8) for t in gpu)), (*want, *(t.view(torch.uint8) for t in mine))):
            assert torch.equal(a, b)


def _norm_leaves(seed):
    g = torch.Generator().manual_seed(seed)
    return [t.cuda() for t in (torch.randn(2, 40, 4, 64, generator=g).bfloat16(), torch.randn(2, 40, 2, 64, generator=g).bfloat16(),
                               torch.randn(64, generator=g), torch.randn(64, generator=g))]


def test_captured_backward():
    fa = _fa()
    cos, sin = (t.cuda() for t in _tables(40, 64))
    base, dys = _norm_leaves(70), [t.detach() for t in _norm_leaves(71)[:2]]

    def step(leaves):
        return torch.autograd.grad(fa.qk_norm_rotary_func(*leaves, cos, sin), leaves, dys)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone().requires_grad_() for t in base])
    torch.cuda.current_stream().wait_stream(side)
    leaves = [t.clone().requires_grad_() for t in base]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grads = step(leaves)
    for turn in range(4):
        with torch.no_grad():
            for t in leaves:
                t.mul_(1.25).add_(0.1)
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, want):
            assert torch.equal(a, b)


def test_capture_with_gradients_while_an_eager_graph_holds_a_leaf_is_refused():
    fa = _fa()
    cos, sin = (t.cuda() for t in _tables(40, 64))
    leaves = [t.requires_grad_() for t in _norm_leaves(72)]
    eager = fa.qk_norm_rotary_func(*leaves, cos, sin)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop it before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fa.qk_norm_rotary_func(*leaves, cos, sin)
    with torch.no_grad():                                        # without gradients nothing stands against it
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fa.qk_norm_rotary_func(*leaves, cos, sin)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, eager))
    first = torch.autograd.grad(eager, leaves, [torch.ones_like(o) for o in eager])
    del eager
    ones = [torch.ones_like(o) for o in out]
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        grads = torch.autograd.grad(fa.qk_norm_rotary_func(*leaves, cos, sin), leaves, ones)
    for _ in range(3):
        g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, first))


def test_capture_of_views_of_a_held_leaf_is_refused():
    """The same where the leaf comes as a view: ragged q and k, a slice of a packed projection."""
    fa = _fa()
    cos, sin = (t.cuda() for t in _tables(40, 64))
    base = _norm_leaves(75)
    w = base[2:]
    pos = torch.arange(40, dtype=torch.int32).cuda()
    flat = [t[0].clone().requires_grad_() for t in base[:2]]
    packed = torch.cat(base[:2], 2)[0].clone().requires_grad_()
    for q, k in ((flat[0], flat[1]), (flat[0], base[1][0]), (base[0][0], flat[1]), (packed[:, :4], packed[:, 4:])):
        eager = fa.qk_norm_rotary_func(q, k, *w, cos, sin, positions=pos)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="drop it before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fa.qk_norm_rotary_func(q, k, *w, cos, sin, positions=pos)
        del eager, q, k
    # an input that an eager operation made
    q = base[0][0].clone().requires_grad_() * 2
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop it before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fa.qk_norm_rotary_func(q, base[1][0], *w, cos, sin, positions=pos)
    del q

    # dropped: captured and right
    def step():
        out = fa.qk_norm_rotary_func(packed[:, :4], packed[:, 4:], *w, cos, sin, positions=pos)
        return torch.autograd.grad(out, packed, [torch.ones_like(o) for o in out])[0]

    want = step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_gradient_of_a_gradient_is_refused():
    leaves = [t.requires_grad_() for t in _norm_leaves(73)]
    out = _fa().qk_norm_rotary_func(*leaves, *(t.cuda() for t in _tables(40, 64)))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out[0].sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out = _fa().qk_norm_rotary_func(*leaves, *(t.cuda() for t in _tables(40, 64)))
        with torch.no_grad():
            leaves[0].mul_(2)
        out[0].sum().backward()


def test_on_another_stream():
    s = _decode_state(74)
    want = _decode_step(_copy(s))
    mine = _copy(s)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):                   # (work in front, so that a launch on the wrong stream would come too early)
            mine["x"] = mine["x"].float().mul(2.0).bfloat16().float().mul(0.5).bfloat16()
        out = _decode_step(mine)
    stream.synchronize()
    assert torch.equal(out, want)


def test_two_streams_at_once():
    """Calls in flight together, split over the keys and merged, share nothing."""
    states = [_decode_state(76), _decode_state(77)]
    want = [_decode_step(_copy(s)) for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    copies = [[_copy(s) for _ in range(10)] for s in states]
    torch.cuda.synchronize()
    outs = [[], []]
    for turn in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(_decode_step(copies[i][turn]))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


# rows = query positions x heads of a group: 1024 at head dims up to 128 and 192 above go through the cache read back
LONG = [
    (2, 300, 8, 2, 128, 16, 32, [700, 300], 0),
    (1, 260, 4, 1, 64, 32, 0, [900], 2),
    (2, 1100, 2, 2, 80, 16, 16, [1100, 1300], 0),
    (2, 200, 2, 2, 256, 16, 64, [333, 201], 0),
    (1, 70, 6, 2, 192, 16, 16, [1000], 3),
    (2, 200, 8, 1, 96, 16, 48, [100, 0], 0),                     # fewer keys than queries, and none
    (1, 40, 6, 2, 256, 16, 16, [999], 0),                        # the same head dim under the limit
    (2, 100, 8, 2, 128, 16, 32, [700, 300], 3),                  # and rows under it
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal,window,alibi", [(False, (-1, -1), False), (True, (-1, -1), True), (False, (100, 7), False)])
@pytest.mark.parametrize("b,sq,h,hk,d,blk,page,lens,num_splits", LONG)
def test_long_queries(b, sq, h, hk, d, blk, page, lens, num_splits, causal, window, alibi, dtype):
    cache = Cache(b, max(lens) + 9, hk, d, blk, page, seed=80)
    slopes = torch.rand(b, h, generator=torch.Generator().manual_seed(81)) * 0.3 if alibi else None
    _check(cache, lens, _q((b, sq, h, d), dtype, 82), dtype, causal=causal, window=window, slopes=slopes, num_splits=num_splits)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("h,hk,d,page,counts,lens", [
    (8, 2, 128, 64, [1, 300, 4, 0, 5, 129], [500, 310, 4, 50, 37, 129]),     # 5 and 0 positions: 20 rows, none
    (2, 2, 256, 32, [201, 16, 17, 1], [222, 400, 17, 3]),
    (40, 1, 64, 16, [30, 1, 2], [90, 300, 2]),                               # more than 32 heads a group
    (72, 1, 64, 16, [20, 1, 0, 3], [90, 300, 7, 3]),                         # more than 64: one position is a long query
])
def test_long_and_short_queries_in_one_batch(h, hk, d, page, counts, lens, dtype):
    cache = Cache(len(lens), max(lens), hk, d, 16, page, seed=83)
    _check(cache, lens, _q((sum(counts), h, d), dtype, 84), dtype, ragged=counts, causal=True)


def test_long_append():
    cache = Cache(2, 700, 2, 128, 16, 32, seed=85)
    news = [_q((2, 280, 2, 128), "bf16", 86 + w) for w in range(2)]
    _check(cache, [400, 3], _q((2, 280, 8, 128), "bf16", 88), "bf16", causal=True, news=news)


@pytest.mark.parametrize("h", [33, 65, 130])
def test_many_heads_on_one_kv_head(h):
    cache = Cache(2, 600, 1, 64, 16, 16, seed=89)
    _check(cache, [600, 11], _q((2, 1, h, 64), "bf16", 90), "bf16")


@pytest.mark.parametrize("b,h,hk,d,cap,num_splits", [(70, 2, 1, 64, 900, 0), (150, 2, 1, 64, 700, 5), (65, 4, 4, 128, 300, 0),
                                                     (300, 1, 1, 16, 200, 0), (1, 2, 1, 64, 9000, 128)])
def test_large_and_uneven_batches(b, h, hk, d, cap, num_splits):
    g = torch.Generator().manual_seed(91)
    lens = (cap * torch.rand(b, generator=g) ** 4).int().tolist()
    lens[0] = cap
    cache = Cache(b, cap, hk, d, 16, 32, seed=92)
    _check(cache, lens, _q((b, 1, h, d), "bf16", 93), "bf16", num_splits=num_splits)


@pytest.mark.parametrize("equal", [True, False])
@pytest.mark.parametrize("b,sq,h,hk,d,cap,dtype,page", [
    (150, 1, 4, 4, 128, 1600, "bf16", 32),           # one to two workgroups a sequence
    (300, 1, 4, 4, 128, 1000, "fp16", 0),            # more sequences than workgroups
    (140, 1, 20, 1, 128, 3000, "bf16", 32),          # 32 rows
    (140, 2, 2, 2, 256, 1600, "fp16", 64),
    (600, 1, 4, 4, 112, 700, "bf16", 16),
    (300, 2, 8, 4, 64, 1200, "bf16", 16),            # pairs of heads
])
def test_runs_of_keys_across_sequences(b, sq, h, hk, d, cap, dtype, page, equal):
    """Batches that parts of equal length leave much of the chip idle with: a workgroup then has pieces of several
    sequences.  Some sequences are empty; the result does not depend on the batch that a sequence is in, beyond the
    order of sums."""
    g = torch.Generator().manual_seed(91)
    lens = [cap] * b if equal else (cap * torch.rand(b, generator=g)).int().tolist()
    lens[3] = lens[70] = 0
    cache = Cache(b, cap, hk, d, 16, page, seed=92)
    _check(cache, lens, _q((b, sq, h, d), dtype, 93), dtype)


@pytest.mark.parametrize("h,hk,d,page", [(2, 2, 64, 16), (4, 2, 128, 32), (6, 2, 48, 0), (8, 1, 64, 16), (2, 1, 256, 32)])
def test_short_ragged_queries(h, hk, d, page):
    """Single tokens, a few drafted ones and sequences without a query in one ragged batch: the decode kernel alone."""
    counts, lens = [1, 3, 2, 0, 1, 4, 1], [900, 3, 77, 50, 1, 1500, 0]
    cache = Cache(len(lens), max(lens), hk, d, 16, page, seed=120)
    for num_splits in (0, 1, 4):
        _check(cache, lens, _q((sum(counts), h, d), "bf16", 121), "bf16", ragged=counts, causal=True, num_splits=num_splits)


def test_runs_of_keys_over_a_ragged_batch():
    g = torch.Generator().manual_seed(122)
    counts = torch.randint(0, 4, (160,), generator=g).tolist()
    lens = (1500 * (0.7 + 0.3 * torch.rand(160, generator=g))).int().tolist()
    cache = Cache(160, 1500, 4, 128, 16, 0, seed=123)
    _check(cache, lens, _q((sum(counts), 4, 128), "fp16", 124), "fp16", ragged=counts, causal=True)


@pytest.mark.parametrize("hk,d,b,sq", [(4, 128, 150, 1), (8, 64, 150, 1), (4, 128, 150, 20), (4, 128, 20, 1), (8, 64, 3, 1)])
def test_long_streams(hk, d, b, sq):
    """Pools of more than 512 MiB of codes, whose loads go past the caches: parts and runs, heads alone and in pairs."""
    small = Cache(b, 1600, hk, d, 16, 64, extra_pages=0, seed=125)
    n = small.codes[0].shape[0]
    pool = 260 * 2 ** 20 // (64 * hk * d) + 1
    pool = max(pool, n)
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(126))[:n]
    gpu = []
    for t, dt in ((small.codes[0], torch.float8_e4m3fn), (small.codes[1], torch.float8_e4m3fn), (small.scales[0], torch.float8_e8m0fnu), (small.scales[1], torch.float8_e8m0fnu)):
        big = torch.full((pool, *t.shape[1:]), 127, dtype=torch.uint8, device="cuda")
        big[ids.cuda()] = t.to(torch.uint8).cuda()
        gpu.append(big.view(dt))
    wide = 260 * 2 ** 20 // (b * 64 * hk * d) + 1                       # pages a sequence may have
    table = torch.zeros(b, max(wide, small.per), dtype=torch.int32)
    table[:, :small.per] = ids[small.table.long()].to(torch.int32)
    lens = (1600 * (0.6 + 0.4 * torch.rand(b, generator=torch.Generator().manual_seed(127)))).int().tolist()
    q = _q((b, sq, hk, d), "bf16", 128).cuda()
    out = _fa().flash_attn_with_quantized_kvcache(q, *gpu, cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=table.cuda(), causal=True)
    for i in range(0, b, 1 if b < 10 else 7):
        want, tol = attend_ref(q[i], small.values(0, i, lens[i]), small.values(1, i, lens[i]), True)
        _close(out[i], want, tol, "sequence %d" % i)


def test_runs_of_keys_with_windows_and_new_tokens():
    b, cap = 150, 1600
    lens = (cap * (0.5 + 0.5 * torch.rand(b, generator=torch.Generator().manual_seed(94)))).int().tolist()
    cache = Cache(b, cap + 2, 4, 128, 16, 16, seed=95)
    q = _q((b, 2, 8, 128), "bf16", 96)
    _check(cache, lens, q, "bf16", causal=True, window=(900, 0))
    _check(cache, lens, q, "bf16", causal=True, news=[_q((b, 2, 4, 128), "bf16", 97 + w) for w in range(2)])
    gpu, table = cache.gpu(), cache.block_table()
    args = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=table, causal=True)
    first = _fa().flash_attn_with_quantized_kvcache(q.cuda(), *gpu, **args)
    for _ in range(10):
        assert torch.equal(first, _fa().flash_attn_with_quantized_kvcache(q.cuda(), *gpu, **args))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,sq,h,hk,d,blk,page,lens,window,num_splits", [
    (2, 1, 2, 2, 64, 16, 16, [700, 33], -1, 0),
    (3, 2, 16, 4, 64, 32, 64, [0, 31, 1777], -1, 3),          # 8 rows a head
    (2, 3, 4, 2, 48, 16, 0, [300, 2], 100, 1),                # fewer keys than queries
    (2, 1, 16, 16, 16, 16, 32, [500, 129], 64, 0),
    (1, 1, 42, 6, 64, 48, 48, [5000], -1, 0),                 # 7 rows; 3 pairs
    (2, 2, 10, 2, 64, 16, 16, [400, 60], -1, 0),              # 10 rows: not in pairs
    (2, 1, 3, 3, 64, 16, 16, [400, 60], -1, 0),               # an odd number of heads
])
def test_narrow_heads_in_pairs(b, sq, h, hk, d, blk, page, lens, window, num_splits, dtype):
    cache = Cache(b, max(lens) + 20, hk, d, blk, page, seed=110)
    slopes = torch.rand(h, generator=torch.Generator().manual_seed(111)) * 0.2 if d == 48 else None
    _check(cache, lens, _q((b, sq, h, d), dtype, 112), dtype, causal=True, window=(window, -1), num_splits=num_splits, slopes=slopes)


def test_a_nan_of_one_head_stays_out_of_its_neighbour():
    for num_splits in (1, 3):
        cache = Cache(2, 300, 4, 64, 16, 16, seed=113)
        clean = cache.gpu()
        q = _q((2, 1, 8, 64), "bf16", 114).cuda()
        args = dict(cache_seqlens=torch.tensor([300, 200], dtype=torch.int32).cuda(), block_table=cache.block_table(), num_splits=num_splits)
        want = _fa().flash_attn_with_quantized_kvcache(q, *clean, **args)
        for which, head in ((0, 1), (1, 2), (0, 2), (1, 3)):
            bad = [t.clone() for t in clean]
            pg, row = cache.place(0, 150)
            bad[which].view(torch.uint8)[pg, row, head] = 127
            got = _fa().flash_attn_with_quantized_kvcache(q, *bad, **args)
            hit = torch.zeros(2, 1, 8, dtype=torch.bool)
            hit[0, :, 2 * head:2 * head + 2] = True
            assert torch.isnan(got[hit.cuda()]).all() and torch.equal(got[~hit.cuda()], want[~hit.cuda()])
        scaled = [t.clone() for t in clean]                  # and a NaN scale
        scaled[2].view(torch.uint8)[pg, 0, 1] = 255
        got = _fa().flash_attn_with_quantized_kvcache(q, *scaled, **args)
        assert torch.isnan(got[0, :, 2:4]).all() and torch.equal(got[0, :, 4:], want[0, :, 4:]) and torch.equal(got[:, :, :2], want[:, :, :2])


@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (8, 2, 128), (4, 2, 256), (40, 2, 64)])
def test_caches_with_heads_outside_and_padded_rows(h, hk, d):
    """A pool stored as (pages, heads, rows, headdim + padding): the same result as the plain layout."""
    cache = Cache(3, 400, hk, d, 16, 32, seed=115)
    plain, table = cache.gpu(), cache.block_table()
    q = _q((3, 1, h, d), "fp16", 116).cuda()
    args = dict(cache_seqlens=torch.tensor([400, 0, 77], dtype=torch.int32).cuda(), block_table=table)
    n = plain[0].shape[0]
    other = []
    for t in plain[:2]:
        wide = torch.full((n, hk, 32, d + 16), 127, dtype=torch.uint8, device="cuda")
        wide[..., :d] = t.view(torch.uint8).transpose(1, 2)
        other.append(wide[..., :d].transpose(1, 2).view(torch.float8_e4m3fn))
    for t in plain[2:]:
        other.append(t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e8m0fnu))
    assert torch.equal(_fa().flash_attn_with_quantized_kvcache(q, *other, **args), _fa().flash_attn_with_quantized_kvcache(q, *plain, **args))


def test_scales_at_the_ends_of_their_range():
    """Bytes 0 and 254 (2^-127, 2^127) and 255 (NaN): never written here, but what a cache from elsewhere can hold."""
    fa = _fa()
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    kc = codes.view(1, 16, 1, 16).repeat(4, 1, 1, 1).cuda().view(torch.float8_e4m3fn)
    sc = torch.tensor([0, 1, 254, 255], dtype=torch.uint8).view(4, 1, 1).cuda().view(torch.float8_e8m0fnu)
    k, v = fa.dequantize_kvcache(kc, kc, sc, sc, torch.full((4,), 16, dtype=torch.int32).cuda(), max_seqlen=16)
    val = codes.view(torch.float8_e4m3fn).double()
    for i, e in enumerate((-127, -126, 127)):
        want = (val * 2.0 ** e).to(torch.bfloat16)          # (2^127: all from 2 on overflows to infinity)
        same = (k[i].flatten().cpu() == want) | (torch.isnan(k[i].flatten().cpu()) & torch.isnan(want))
        assert bool(same.all()), (e, codes[~same])
    assert torch.isnan(k[3]).all() and torch.equal(k.view(torch.int16), v.view(torch.int16))
    h, _ = fa.dequantize_kvcache(kc, kc, sc, sc, torch.full((4,), 16, dtype=torch.int32).cuda(), max_seqlen=16, dtype=torch.float16)
    for i, e in enumerate((-127, -126, 127)):               # fp16 holds none of these: zeros and infinities
        want, got = (val * 2.0 ** e).to(torch.float16), h[i].flatten().cpu()
        assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all()), e
    # a token that joins a block at 2^127, and one whose scale is NaN
    x = torch.zeros(4, 1, 1, 16, dtype=torch.bfloat16)
    x[:, :, :, 0] = 2.0 ** 127
    x[:, :, :, 1] = -2.0 ** 118
    fa.quantize_kvcache(x.cuda(), x.cuda(), kc, kc.clone(), sc, sc.clone(), torch.full((4,), 15, dtype=torch.int32).cuda())
    got = kc.view(torch.uint8)[2, 15, 0].cpu().to(torch.int32)
    assert got.tolist() == encode(torch.tensor([1.0, -2.0 ** -9] + [0.0] * 14, dtype=torch.float64)).tolist()
    assert sc.view(torch.uint8)[2:].flatten().tolist() == [254, 255]


def test_attention_offsets_past_32_bits():
    """A pool of more than 4 GiB of codes per tensor, pages at both ends; a contiguous sequence of more than 2^32 bytes,
    its last keys; both with streams that go past the caches."""
    fa = _fa()
    hk, d, rows = 8, 128, 64
    n = 70000                                            # pages of 64 KiB
    kc = torch.zeros(n, rows, hk, d, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.full((n, 4, hk), 122, dtype=torch.uint8, device="cuda")
    vs = torch.full_like(ks, 121)
    small = Cache(2, 300, hk, d, 16, rows, extra_pages=0, seed=94)
    ids = torch.tensor([0, n - 1, 65536, 65535, n // 2, n - 2, 1, 65537, 69000, 68000])
    for t, c in ((kc, small.codes[0]), (vc, small.codes[1]), (ks, small.scales[0]), (vs, small.scales[1])):
        t[ids.cuda()] = c.to(torch.uint8).cuda()
    table = ids[small.table.long()].to(torch.int32).cuda()
    q = _q((2, 1, 16, d), "bf16", 95)
    lens = [300, 190]
    view = (kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn), ks.view(torch.float8_e8m0fnu), vs.view(torch.float8_e8m0fnu))
    out = fa.flash_attn_with_quantized_kvcache(q.cuda(), *view, cache_seqlens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table=table)
    for i, m in enumerate(lens):
        want, tol = attend_ref(q[i].cuda(), small.values(0, i, m), small.values(1, i, m))
        _close(out[i], want, tol, "page %d" % i)
    # the same memory as one sequence of 4.48 million tokens and 4.6e9 bytes
    flat = [t.flatten(0, 1)[None] for t in (kc, vc, ks, vs)]
    total = n * rows
    last = Cache(1, 256, hk, d, 16, 0, seed=96)
    for t, c in ((flat[0], last.codes[0]), (flat[1], last.codes[1])):
        t[0, -256:] = c[0].to(torch.uint8).cuda()
    for t, c in ((flat[2], last.scales[0]), (flat[3], last.scales[1])):
        t[0, -16:] = c[0].to(torch.uint8).cuda()
    flat = [t.view(torch.float8_e4m3fn if i < 2 else torch.float8_e8m0fnu) for i, t in enumerate(flat)]
    q = _q((1, 3, 16, d), "bf16", 97)
    for long_q in (q, _q((1, 100, 16, d), "bf16", 98)):
        out = fa.flash_attn_with_quantized_kvcache(long_q.cuda(), *flat, cache_seqlens=torch.tensor([total], dtype=torch.int32).cuda(),
                                                   causal=True, window_size=(100, 0))
        want, tol = attend_ref(long_q[0].cuda(), last.values(0, 0, 256), last.values(1, 0, 256), True, (100, 0))
        _close(out[0], want, tol, "end of a long sequence")


def test_views_of_weights_tables_and_positions():
    fa = _fa()
    g = torch.Generator().manual_seed(99)
    q, k = (torch.randn(2, 6, n, 64, generator=g).half().cuda() for n in (3, 1))
    w = torch.randn(64, generator=g).half().cuda()
    cos, sin = (t.half().cuda() for t in _tables(20, 64))
    pos = torch.randint(0, 20, (2, 6), generator=g).to(torch.int32).cuda()
    want = fa.qk_norm_rotary_func(q, k, w, w, cos, sin, positions=pos)
    off = torch.empty(65, dtype=torch.float16, device="cuda")[1:]          # not 16-byte aligned
    off.copy_(w)
    tables = []
    for t in (cos, sin):
        tables.append(torch.empty(t.numel() + 3, dtype=torch.float16, device="cuda")[3:].view(t.shape))
        tables[-1].copy_(t)
    wide = torch.empty(2, 6, 2, dtype=torch.int32, device="cuda")
    wide[..., 0] = pos
    odd_q = torch.empty(2, 6, 3, 68, dtype=torch.float16, device="cuda")[..., 1:65]
    odd_q.copy_(q)
    got = fa.qk_norm_rotary_func(odd_q, k, off, w, *tables, positions=wide[..., 0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for bad in (dict(positions=pos.cpu()), dict(positions=pos.long()), dict(positions=pos[:1])):
        with pytest.raises(RuntimeError):
            fa.qk_norm_rotary_func(q, k, w, w, cos, sin, **bad)
    with pytest.raises(RuntimeError):
        fa.qk_norm_rotary_func(q, k.bfloat16(), w, w, cos, sin)
    with pytest.raises(RuntimeError):
        fa.qk_norm_rotary_func(q, k, w.bfloat16(), w.bfloat16(), cos, sin)
    with pytest.raises(RuntimeError):
        fa.qk_norm_rotary_func(q, k, w, w.cpu(), cos, sin)


def test_refusals_with_tensors_on_the_device():
    fa = _fa()
    cache = Cache(2, 64, 2, 64, 16, 16, seed=100)
    kc, vc, ks, vs = cache.gpu()
    table, lens = cache.block_table(), torch.tensor([10, 64], dtype=torch.int32).cuda()
    q, x = _q((2, 1, 4, 64), "bf16", 101).cuda(), _q((2, 1, 2, 64), "bf16", 102).cuda()
    before = [t.view(torch.uint8).clone() for t in (kc, vc, ks, vs)]
    attend = lambda q=q, kc=kc, vc=vc, ks=ks, vs=vs, **kw: fa.flash_attn_with_quantized_kvcache(
        q, kc, vc, ks, vs, **{**dict(cache_seqlens=lens, block_table=table), **kw})
    for call in (
        lambda: attend(cache_seqlens=lens.cpu()), lambda: attend(cache_seqlens=lens.long()), lambda: attend(cache_seqlens=lens[:1]),
        lambda: attend(block_table=table.cpu()), lambda: attend(block_table=table[:1]), lambda: attend(cache_batch_idx=lens),
        lambda: attend(q=q.float()), lambda: attend(q=q[..., :32]), lambda: attend(q=_q((2, 1, 3, 64), "bf16", 0).cuda()),
        lambda: attend(ks=ks[:, :, :1]), lambda: attend(ks=ks.view(torch.uint8)), lambda: attend(kc=kc.view(torch.uint8)),
        lambda: attend(kc=kc[:, :8], vc=vc[:, :8]), lambda: attend(vs=vs[:-1]), lambda: attend(k=x), lambda: attend(k=x, v=x, cache_seqlens=None),
        lambda: attend(k=x.half(), v=x.half()), lambda: attend(k=x[:1], v=x[:1]), lambda: attend(softmax_scale=0.0), lambda: attend(num_splits=129),
        lambda: attend(softmax_scale=-1.0), lambda: attend(out=q.float()), lambda: attend(out=q[:1]), lambda: attend(q=q.cpu()),
        lambda: attend(q=q[:, 0], cu_seqlens_q=torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), max_seqlen_q=1, k=x, v=x),
        lambda: fa.quantize_kvcache(x.float(), x.float(), kc, vc, ks, vs, lens, block_table=table),
        lambda: fa.quantize_kvcache(x, x[..., :48], kc, vc, ks, vs, lens, block_table=table),
        lambda: fa.quantize_kvcache(x[:, :, :1], x[:, :, :1], kc, vc, ks, vs, lens, block_table=table),
        lambda: fa.dequantize_kvcache(kc, vc, ks, vs, lens, max_seqlen=-1, block_table=table),
        lambda: fa.dequantize_kvcache(kc, vc, ks, vs, lens, max_seqlen=4, block_table=table, dtype=torch.float32),
    ):
        with pytest.raises(RuntimeError):
            call()
    for a, b in zip(before, (kc, vc, ks, vs)):           # refused before anything was written
        assert torch.equal(a, b.view(torch.uint8))
    # no query, and no new tokens: nothing to do, the cache left alone
    assert attend(q=q[:, :0]).shape == (2, 0, 4, 64)
    assert torch.equal(attend(k=x[:, :0], v=x[:, :0]), attend())
    for a, b in zip(before, (kc, vc, ks, vs)):
        assert torch.equal(a, b.view(torch.uint8))
    # no query, but new tokens: written
    attend(q=q[:, :0], k=x, v=x)
    assert not torch.equal(before[0], kc.view(torch.uint8))


def test_a_padded_batch_writes_nothing_for_its_padding():
    """Sequences whose table (or batch index) names no page: their tokens are dropped, the pool stays as it is."""
    for page in (16, 0):
        cache = Cache(3, 64, 2, 64, 16, page, seed=103)
        gpu = cache.gpu()
        rows_of = None if page else torch.tensor([2, -1, 1], dtype=torch.int32)
        table = None
        if page:
            table = cache.table.clone()
            table[1] = -1
            table = table.cuda()
        lens = torch.tensor([5, 0, 20], dtype=torch.int32).cuda()
        q, x = _q((3, 1, 4, 64), "bf16", 104).cuda(), _q((3, 1, 2, 64), "bf16", 105)
        out = _fa().flash_attn_with_quantized_kvcache(q, *gpu, k=x.cuda(), v=x.cuda(), cache_seqlens=lens, block_table=table,
                                                      cache_batch_idx=None if rows_of is None else rows_of.cuda())
        for i in (0, 2):
            for w in range(2):
                write_ref(cache, w, i, int(lens[i]), x[i], "bf16", rows_of)
        for t, want in zip(gpu, (*cache.codes, *cache.scales)):
            assert torch.equal(t.view(torch.uint8).cpu().to(torch.int32), want)
        assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
