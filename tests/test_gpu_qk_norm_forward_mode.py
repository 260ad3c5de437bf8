"""qk_norm_rotary_func has no forward-mode derivative: an input with a tangent is refused, not taken for a constant."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_a_tangent_is_refused(which, requires_grad):
    import vllm_flash_attn as fa
    g = torch.Generator().manual_seed(230)
    a = [torch.randn(s, generator=g).cuda() for s in ((1, 5, 4, 64), (1, 5, 2, 64), (64,), (64,), (5, 16), (5, 16))]
    a = [x.bfloat16() if i < 2 else x for i, x in enumerate(a)]
    if requires_grad:
        a[1].requires_grad_()
    plain = fa.qk_norm_rotary_func(*a)
    with fwAD.dual_level():
        b = list(a)
        b[which] = fwAD.make_dual(a[which].detach(), torch.ones_like(a[which]))
        with pytest.raises(RuntimeError, match="forward"):
            fa.qk_norm_rotary_func(*b)
        for x, y in zip(fa.qk_norm_rotary_func(*a), plain):        # without a tangent nothing stands against it
            assert torch.equal(x, y)
