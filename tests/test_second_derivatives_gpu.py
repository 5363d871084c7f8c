"""The differentiable operators have first derivatives only. A second one raises, along whichever path it is asked for -
also where PyTorch would take a missing path for a derivative of zero."""
import pytest
import torch

from paraattention_b200 import ops

pytestmark = pytest.mark.gpu


def cross():
    g = torch.Generator(device="cuda").manual_seed(0)
    xs = [torch.randn(2, 2, s, 64, device="cuda", generator=g).bfloat16().requires_grad_(True) for s in (130, 40, 40)]
    return ops.cross_attention(*xs), xs


def norm():
    g = torch.Generator(device="cuda").manual_seed(0)
    xs = [torch.randn(2, 2, 30, 64, device="cuda", generator=g).bfloat16().requires_grad_(True) for _ in range(2)]
    ws = [torch.ones(64, device="cuda").bfloat16().requires_grad_(True) for _ in range(2)]
    y = ops.qk_norm_rotary(*xs, *ws)
    return y[0], [xs[0], ws[0]]


@pytest.mark.parametrize("make", [cross, norm])
def test_every_path_to_a_second_derivative_raises(make):
    out, xs = make()
    do = torch.randn_like(out).requires_grad_(True)
    first = torch.autograd.grad(out, xs, do, create_graph=True)
    for g in first:
        for source in (*xs, do):
            with pytest.raises(RuntimeError, match="once"):
                torch.autograd.grad(g.float().square().sum(), source, allow_unused=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            g.float().sum().backward(retain_graph=True)


@pytest.mark.parametrize("make", [cross, norm])
def test_recording_the_backward_pass_is_no_error(make):
    out, xs = make()
    do = torch.randn_like(out)
    recorded = torch.autograd.grad(out, xs, do, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(recorded, torch.autograd.grad(out, xs, do)))


def test_forward_derivatives_by_a_second_backward_pass():
    from torch.autograd.functional import hvp, jvp

    _, (q, k, v) = cross()
    k, v = k.detach(), v.detach()
    with pytest.raises(RuntimeError, match="once"):
        jvp(lambda x: ops.cross_attention(x, k, v), q.detach(), torch.ones_like(q))
    with pytest.raises(RuntimeError, match="once"):
        hvp(lambda x: ops.cross_attention(x, k, v).float().square().sum(), q.detach(), torch.ones_like(q))
    with pytest.raises(RuntimeError, match="once"):
        jvp(lambda x: ops.qk_norm_rotary(x)[0], q.detach(), torch.ones_like(q))
