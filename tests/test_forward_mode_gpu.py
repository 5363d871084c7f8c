"""The differentiable operators compute no forward-mode derivatives, and say so instead of dropping a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from paraattention_b200 import ops

pytestmark = pytest.mark.gpu


def make(B=2, H=2, Sq=200, Skv=150, D=64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, s, H, D, device="cuda", generator=g).bfloat16().transpose(1, 2) for s in (Sq, Skv, Skv)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("Sq", [1, 200])
def test_cross_attention_refuses_forward_mode(Sq, which, grad):
    xs = [t.requires_grad_(grad) for t in make(Sq=Sq)]
    with fwAD.dual_level():
        xs[which] = fwAD.make_dual(xs[which], torch.ones_like(xs[which]))
        with pytest.raises(NotImplementedError, match="jvp|forward"):
            ops.cross_attention(*xs)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            ops.cross_attention(*xs)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_norm_refuses_forward_mode(which, grad):
    q, k, _ = make(Skv=200)
    xs = [t.requires_grad_(grad) for t in (q, k, torch.ones_like(q[0, 0, 0]), torch.ones_like(q[0, 0, 0]))]
    with fwAD.dual_level():
        xs[which] = fwAD.make_dual(xs[which], torch.ones_like(xs[which]))
        with pytest.raises(NotImplementedError, match="jvp|forward"):
            ops.qk_norm_rotary(*xs)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            ops.qk_norm_rotary(*xs)


def test_norm_refuses_forward_mode_of_the_tables():
    q, _, _ = make()
    cos, sin = torch.ones(200, 64, device="cuda"), torch.zeros(200, 64, device="cuda")
    with fwAD.dual_level():
        for tables in ((fwAD.make_dual(cos, cos), sin), (cos, fwAD.make_dual(sin, cos))):
            with pytest.raises(NotImplementedError, match="forward"):
                ops.qk_norm_rotary(q, None, None, None, tables)


def test_backward_passes_refuse_forward_mode():
    """Output gradients with a tangent: the backward passes are functions of them, too."""
    q, k, v = (t.requires_grad_(True) for t in make())
    out = ops.cross_attention(q, k, v)
    y, _ = ops.qk_norm_rotary(q, None, torch.ones_like(q[0, 0, 0]).detach())
    do = torch.ones_like(out)
    with fwAD.dual_level():
        dual = fwAD.make_dual(do, do.clone())
        for o, xs in ((out, (q, k, v)), (y, (q,))):
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(o, xs, dual, retain_graph=True)
            assert all(g.isfinite().all() for g in torch.autograd.grad(o, xs, do, retain_graph=True))


def test_what_the_dual_level_leaves_alone_goes_through():
    """Inside a dual level, tensors without a tangent are ordinary ones."""
    q, k, v = make()
    want = ops.cross_attention(q, k, v)
    with fwAD.dual_level():
        assert torch.equal(ops.cross_attention(q, k, v), want)
        dual = fwAD.make_dual(q, torch.ones_like(q))
        with fwAD._set_fwd_grad_enabled(False):  # as inside the forward of a function with a rule of its own
            assert torch.equal(ops.cross_attention(dual, k, v), want)
