"""qk_norm_rotary_func, forward and backward, against the formula in 64 bits and against differences."""
import pytest
import torch

from kv8_util import HALF_STEP, TDT, norm_rotary_ref

pytestmark = pytest.mark.gpu


def _fa():
    import vllm_flash_attn as fa
    return fa


def _tables(rows, rd, dtype):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    return a.cos().to(dtype), a.sin().to(dtype)


def _reference(x, w, cos, sin, pos, dy, eps, inter):
    """out, dx, dw in 64 bits and how far fp32 arithmetic with one rounding may be off, element by element."""
    ok = (pos >= 0)[..., None]
    at = pos.clamp_min(0).long()
    c, s = cos.double()[at], sin.double()[at]
    x = x.double().requires_grad_()
    w = w.double().requires_grad_()
    y = norm_rotary_ref(x, w, c, s, pos, eps, inter)
    y = torch.where(ok[..., None], y, 0.0)
    dx, dw = torch.autograd.grad(y, (x, w), dy.double())
    return y.detach(), dx, dw


# b, s, h, hk, d, rd, interleaved, table, weight
SHAPES = [
    (1, 1, 1, 1, 16, 16, False, "fp32", "same"),
    (2, 3, 4, 2, 64, 64, True, "same", "same"),
    (1, 37, 7, 1, 128, 128, False, "fp32", "fp32"),
    (3, 5, 8, 8, 80, 32, False, "same", "same"),
    (2, 9, 5, 3, 96, 64, True, "fp32", "same"),
    (1, 130, 3, 2, 256, 256, False, "same", "fp32"),
    (2, 11, 2, 1, 200, 112, False, "fp32", "same"),
    (1, 6, 33, 17, 24, 16, True, "same", "same"),
    (1, 1025, 4, 4, 192, 192, True, "fp32", "same"),
    (4, 1, 32, 8, 128, 64, False, "same", "same"),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,s,h,hk,d,rd,inter,table,weight", SHAPES)
@pytest.mark.parametrize("given", [False, True])
def test_forward_and_gradients(b, s, h, hk, d, rd, inter, table, weight, given, dtype):
    g = torch.Generator().manual_seed(1)
    dt, u, eps = TDT[dtype], HALF_STEP[dtype], 1e-5
    wt = torch.float32 if weight == "fp32" else dt
    cos, sin = _tables(max(s, 50), rd, torch.float32 if table == "fp32" else dt)
    pos = torch.randint(0, cos.shape[0], (b, s), generator=g).to(torch.int32) if given else torch.arange(s).expand(b, s).to(torch.int32)
    if given:
        pos[0, s // 2] = -1 if b * s > 1 else pos[0, s // 2]     # a padded token
    packed = (torch.randn(b, s, (h + hk) * d + 8, generator=g) * torch.exp(torch.randn(b, s, 1, generator=g))).to(dt)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g)).to(wt) for _ in range(2))
    dys = [torch.randn(b, s, n, d, generator=g).to(dt) for n in (h, hk)]
    dev = packed.cuda()
    q = dev[..., :h * d].view(b, s, h, d).detach().requires_grad_()
    k = dev[..., h * d:(h + hk) * d].view(b, s, hk, d).detach().requires_grad_()
    gw = [w.cuda().requires_grad_() for w in (wq, wk)]
    out = _fa().qk_norm_rotary_func(q, k, *gw, cos.cuda(), sin.cuda(), positions=pos.cuda() if given else None, eps=eps,
                                    rotary_interleaved=inter)
    grads = torch.autograd.grad(out, (q, k, *gw), [y.cuda() for y in dys])
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        y, dx, dw = _reference(x.detach().cpu(), w, cos, sin, pos, dys[i], eps, inter)
        # fp32: the row's sum of squares (d terms) and about ten more operations; a turned element is a sum of two
        # products, each as large as the pair allows; fp16 can be subnormal
        f32 = (d + 12) * 2.0 ** -24
        floor = 2.0 ** -25 if dtype == "fp16" else 0.0
        r = 1 / (x.detach().cpu().double().square().mean(-1, keepdim=True) + eps).sqrt()
        n = (x.detach().cpu().double() * r * w.double()).abs()
        pair = n.amax(-1, keepdim=True) * 2
        got = out[i].detach().cpu().double()
        assert bool(((got - y).abs() <= u * y.abs() + f32 * pair + floor).all())
        # dx = r (g w - x r mean(g w x r)): terms up to r |dy| |w| and the mean's, each with that error
        gmax = dys[i].double().abs().amax(-1, keepdim=True) * 2 * w.double().abs().max()
        xr = (x.detach().cpu().double() * r).abs()
        size = r * (gmax + xr * (gmax * xr.mean(-1, keepdim=True)))
        gx = grads[i].cpu().double()
        assert bool(((gx - dx).abs() <= u * dx.abs() + 2 * f32 * size + floor).all())
        # dw: a sum over b s heads terms of at most |dy pair| |x r|, in fp32
        terms = b * s * x.shape[2]
        reach = (gmax / w.double().abs().max() * xr).sum((0, 1, 2))
        uw = u if weight == "same" else 2.0 ** -24
        gwt = grads[2 + i].cpu().double()
        assert grads[2 + i].dtype == wt
        assert bool(((gwt - dw).abs() <= uw * dw.abs() + (terms + d + 12) * 2.0 ** -24 * reach + floor).all())
        if given and b * s > 1:
            assert not out[i][0, s // 2].any() and not grads[i][0, s // 2].any()


def test_gradients_against_differences():
    """Directional differences of the formula in 64 bits at the 16-bit inputs, along random directions."""
    g = torch.Generator().manual_seed(2)
    b, s, h, hk, d, rd = 1, 6, 2, 1, 32, 16
    cos, sin = _tables(s, rd, torch.float32)
    x = [torch.randn(b, s, n, d, generator=g).to(torch.float16) for n in (h, hk)]
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(torch.float16) for _ in range(2)]
    dys = [torch.randn(b, s, n, d, generator=g).to(torch.float16) for n in (h, hk)]
    leaves = [t.cuda().requires_grad_() for t in (*x, *w)]
    out = _fa().qk_norm_rotary_func(*leaves, cos.cuda(), sin.cuda(), rotary_interleaved=False)
    grads = torch.autograd.grad(out, leaves, [y.cuda() for y in dys])
    pos = torch.arange(s).expand(b, s)

    def loss(args):
        return sum(float((norm_rotary_ref(args[i], args[2 + i], cos.double()[pos], sin.double()[pos], pos, 1e-6, False) * dys[i].double()).sum())
                   for i in range(2))

    base = [t.detach().cpu().double() for t in leaves]
    for i, t in enumerate(base):
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        step = 1e-5
        hi, lo = ([a + s_ * step * v if j == i else a for j, a in enumerate(base)] for s_ in (1, -1))
        want = (loss(hi) - loss(lo)) / (2 * step)
        got = float((grads[i].cpu().double() * v).sum())
        # every gradient element is rounded once to fp16; the difference itself is good to about 1e-7
        tol = float((grads[i].cpu().double().abs() * v.abs()).sum()) * 2.0 ** -11 * 1.1 + 1e-5
        assert abs(got - want) <= tol, (i, got, want, tol)


def test_some_gradients_only_and_odd_gradient_layouts():
    g = torch.Generator().manual_seed(3)
    dev = "cuda"
    q, k = (torch.randn(2, 5, n, 64, generator=g).to(dev, torch.bfloat16) for n in (4, 2))
    wq, wk = (torch.ones(64, device=dev, dtype=torch.bfloat16) for _ in range(2))
    cos, sin = (t.to(dev) for t in _tables(5, 64, torch.float32))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    out = _fa().qk_norm_rotary_func(*leaves, cos, sin)
    full = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    # a gradient that is a broadcast scalar, as sum() gives it
    out = _fa().qk_norm_rotary_func(*leaves, cos, sin)
    same = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)
    for a, b in zip(full, same):
        assert torch.equal(a, b)
    # each leaf alone; one output alone
    for i in range(4):
        args = [t if j != i else t.clone().requires_grad_() for j, t in enumerate((q, k, wq, wk))]
        out = _fa().qk_norm_rotary_func(*args, cos, sin)
        (got,) = torch.autograd.grad(out, args[i], [torch.ones_like(o) for o in out])
        assert torch.equal(got, full[i])
    out = _fa().qk_norm_rotary_func(*leaves, cos, sin)
    dq, dk, dwq, dwk = torch.autograd.grad(out[0].sum(), leaves, allow_unused=True)
    assert torch.equal(dq, full[0]) and torch.equal(dwq, full[2]) and not dk.any() and not dwk.any()
    # the same heads for every query head (a broadcast input): its gradient is the sum over the heads
    one = q[:, :, :1].clone().requires_grad_()
    out = _fa().qk_norm_rotary_func(one.expand(2, 5, 4, 64), k, wq, wk, cos, sin)
    (got,) = torch.autograd.grad(out[0].float().sum(), one)
    each = torch.autograd.grad(_fa().qk_norm_rotary_func(one, k, wq, wk, cos, sin)[0].float().sum(), one)[0]
    # four equal bf16 gradients, added in fp32 or in bf16 (three roundings): 4 * each exactly, or within 3 half steps
    assert bool(((got.float() - 4 * each.float()).abs() <= 3 * 2.0 ** -8 * 4 * each.float().abs()).all())


def test_ragged_form_positions_past_the_table_and_empty():
    g = torch.Generator().manual_seed(4)
    dev = "cuda"
    q, k = (torch.randn(7, n, 128, generator=g).to(dev, torch.float16) for n in (4, 1))
    w = torch.ones(128, device=dev)
    cos, sin = (t.to(dev) for t in _tables(20, 64, torch.float32))
    pos = torch.tensor([0, 1, 2, 0, 19, 20, -3], dtype=torch.int32, device=dev)
    a = _fa().qk_norm_rotary_func(q, k, w, w, cos, sin, positions=pos)
    b = _fa().qk_norm_rotary_func(q[None], k[None], w, w, cos, sin, positions=pos[None])
    for x, y in zip(a, b):
        assert x.dim() == 3 and torch.equal(x.nan_to_num(9.0), y[0].nan_to_num(9.0))
        assert torch.isnan(x[5, :, :64]).all() and torch.isfinite(x[5, :, 64:]).all()      # row 20 of 20
        assert not x[6].any() and torch.isfinite(x[:5]).all()
    leaves = [t.requires_grad_() for t in (torch.empty(0, 3, 2, 64, device=dev, dtype=torch.bfloat16), torch.empty(0, 3, 1, 64, device=dev, dtype=torch.bfloat16),
                                           torch.ones(64, device=dev), torch.ones(64, device=dev))]
    out = _fa().qk_norm_rotary_func(*leaves, *(t.to(dev) for t in _tables(3, 64, torch.float32)))
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    assert out[0].shape == (0, 3, 2, 64) and not grads[2].any() and not grads[3].any()


def test_gradients_are_bitwise_reproducible():
    g = torch.Generator().manual_seed(5)
    leaves = [t.cuda().requires_grad_() for t in (torch.randn(2, 700, 8, 128, generator=g).bfloat16(), torch.randn(2, 700, 2, 128, generator=g).bfloat16(),
                                                  torch.randn(128, generator=g), torch.randn(128, generator=g))]
    cos, sin = (t.cuda() for t in _tables(700, 128, torch.float32))
    dys = [torch.randn(2, 700, n, 128, generator=g).bfloat16().cuda() for n in (8, 2)]
    runs = [torch.autograd.grad(_fa().qk_norm_rotary_func(*leaves, cos, sin), leaves, dys) for _ in range(10)]
    for r in runs[1:]:
        for a, b in zip(runs[0], r):
            assert torch.equal(a, b)
