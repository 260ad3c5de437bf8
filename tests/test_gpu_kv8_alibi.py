"""ALiBi over a long 8-bit KV cache: the bias of the keys that count is small, so must be the scores' error, whatever the
position; and the log-sum-exp that the C ABI writes."""
import pytest
import torch

from kv8_util import HALF_STEP, Cache
from test_gpu_kv8_attention import _close, _q

pytestmark = pytest.mark.gpu


def _reference(q, k, v, slope, causal):
    """64 bits: out, row sums of p |v|, log-sum-exp and the scores' largest magnitude; q (m, h, d), k / v (n, hk, d)."""
    (m, h, d), n = q.shape, k.shape[0]
    r = h // k.shape[1]
    i, j = torch.arange(m, device=q.device)[:, None] + n - m, torch.arange(n, device=q.device)[None]
    outs = []
    for a in range(h):
        kk, vv = k[:, a // r].to(q.device), v[:, a // r].to(q.device)
        s = q[:, a].double() @ kk.t().contiguous() * d ** -0.5
        top = float(s.abs().max())
        s = s - slope * (i - j).abs()
        if causal:
            s = s.masked_fill(j > i, -torch.inf)
        p = torch.softmax(s, 1)
        outs.append((p @ vv, p @ vv.abs(), torch.logsumexp(s, 1), top))
    return [torch.stack([o[x] for o in outs], 1) for x in range(3)] + [max(o[3] for o in outs)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("num_splits", [0, 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("sq,h,hk,d", [(1, 8, 2, 128), (4, 4, 4, 64), (100, 2, 1, 128)])
def test_far_positions(sq, h, hk, d, causal, num_splits, dtype):
    """A score's error, in units of 2^-24: its product of d terms, d * scale sum |q||k|; its bias and the sum with it, three
    times their size, which is at most 40 + 3 top for the keys that count (the others have p < 2^-57).  In fp16 a P under 2^-14 is
    off by up to 2^-25 of the row's largest, of (40 + 3 top) / slope keys on either side."""
    import vllm_flash_attn_2_cuda as E
    slope, n = 0.5, 60000
    cache = Cache(1, n, hk, d, 64, 64, seed=260)
    for s in cache.scales:
        s.fill_(127 - 7)
    q = _q((1, sq, h, d), dtype, 261).cuda()
    out, lse = E.fwd_kv8(q, *cache.gpu(), None, None, torch.tensor([n], dtype=torch.int32).cuda(), None, cache.block_table(),
                         torch.full((h,), slope).cuda(), None, None, 0, d ** -0.5, causal, -1, -1, num_splits)
    k, v = cache.values(0, 0, n), cache.values(1, 0, n)
    want, reach, want_lse, top = _reference(q[0], k, v, slope, causal)
    size = float((q[0].double().abs().amax(0).amax(0) * d ** -0.5).sum()) * float(k.abs().max())
    ds = 2.0 ** -24 * (d * size + 3 * (40 + 3 * top)) + 2.0 ** -20
    u = HALF_STEP[dtype]
    tol = u * want.abs() + (u + 2 * ds) * (1 + 4 * u) * reach
    if dtype == "fp16":
        tol = tol + (2 * (40 + 3 * top) / slope * float(v.abs().max()) + 1) * 2.0 ** -25
    _close(out[0], want, tol)
    # (the log-sum-exp: its own few roundings beside the scores' error)
    assert bool(((lse[0].t().double() - want_lse).abs() <= ds + 2.0 ** -22 * (want_lse.abs() + top + 20)).all())
    # an error of two roundings, that does not grow with the position (2^-24 * slope * n would be 1.8e-3)
    e = float((out[0].double() - want).norm() / want.norm())
    assert e <= u, "relative error %.2e" % e
