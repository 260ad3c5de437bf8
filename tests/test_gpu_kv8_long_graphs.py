"""Long queries over an 8-bit KV cache (chunks over the codes, over the cache read back, with the keys in parts, ragged batches
of chunks and single tokens) captured into graphs, and on two streams at once: what the launches of a call hand to each
other lies in a workspace of the call's own."""
import pytest
import torch

from kv8_util import Cache
from test_gpu_kv8_attention import _q

pytestmark = pytest.mark.gpu

#        counts (ragged) or (b, sq), h, hk, d, num_splits, window
CALLS = [((2, 100), 8, 2, 128, 0, (-1, -1)), ((2, 300), 8, 2, 128, 0, (-1, -1)), ((1, 270), 8, 2, 96, 3, (-1, -1)), ((2, 100), 4, 2, 256, 0, (-1, -1)),
         ((2, 200), 4, 2, 256, 2, (60, 0)), ([1, 300, 4, 1], 8, 2, 128, 0, (-1, -1)), ([200, 1, 0, 5], 4, 2, 256, 0, (90, -1))]


def _state(call, seed):
    shape, h, hk, d, num_splits, window = call
    ragged = isinstance(shape, list)
    b = len(shape) if ragged else shape[0]
    cache = Cache(b, 1000, hk, d, 16, 32, seed=seed)
    lens = torch.tensor([[600, 811, 333, 702][i] for i in range(b)], dtype=torch.int32).cuda()
    kw = dict(cache_seqlens=lens, block_table=cache.block_table(), causal=window[0] < 0, window_size=window, num_splits=num_splits)
    if ragged:
        kw.update(cu_seqlens_q=torch.tensor([0] + shape).cumsum(0).to(torch.int32).cuda(), max_seqlen_q=max(shape))
    q = _q((sum(shape), h, d) if ragged else (*shape, h, d), "bf16", seed + 1).cuda()
    return q, cache.gpu(), kw


def _call(state):
    import vllm_flash_attn as fa
    q, gpu, kw = state
    return fa.flash_attn_with_quantized_kvcache(q, *gpu, **kw)


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_two_graphs_replayed_in_turn(call):
    states = [_state(call, 270), _state(call, 280)]
    for s in states:
        _call(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(_call(s))
        graphs.append(g)
    for turn in range(4):
        want = []
        for q, gpu, kw in states:
            q.mul_(-1.25)
            kw["cache_seqlens"].add_(29 * turn)
            want.append(_call((q, gpu, kw)))
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i]), (turn, i)


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_two_streams_at_once(call):
    states = [_state(call, 290), _state(call, 300)]
    want = [_call(s) for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(_call(states[i]))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
