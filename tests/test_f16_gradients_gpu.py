"""Gradients of ops.cross_attention in f16 over the range of output gradients: f16's smallest steps are absolute
(2^-24), so what the backward kernel rounds on the way (P and dS) must not come near them while the results are
far from them, and must not pass f16's largest value while the results fit.

Bounds: those of block_ops_reference.py - relative roundings and absolute sums - plus the results' own smallest half
step, 2^-25, and nothing else. Why the terms below cover a scaled dS: the largest it could be is
kept between 2^14 and 2^15 and its smallest half step is 2^-25, that is at most 2^-39 of that largest for each key, far below
SLACK = 2^-13 of the row's sums."""
import math

import pytest
import torch

from block_ops_reference import assert_within, cross_reference
from paraattention_b200 import ops

pytestmark = pytest.mark.gpu

HALF_STEP = 2.0 ** -25


def make(B, Hq, Hkv, Sq, Skv, D, do_size, seed=0, kv_batch=None, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(b, s, h, size=1.0):
        return (torch.randn(b, s, h, D, device="cuda", generator=g) * size).to(dtype).transpose(1, 2)

    kb = B if kv_batch is None else kv_batch
    leaves = [x.requires_grad_(True) for x in (t(B, Sq, Hq), t(kb, Skv, Hkv), t(kb, Skv, Hkv))]
    return (*leaves, t(B, Sq, Hq, do_size))


def check(q, k, v, do, mask=None, what="", asked=(0, 1, 2)):
    xs = [x if i in asked else x.detach() for i, x in enumerate((q, k, v))]
    grads = torch.autograd.grad(ops.cross_attention(*xs, mask), [xs[i] for i in asked], do)
    want, bound = cross_reference(q, k, v, mask, None, do)
    for i, got in zip(asked, grads):
        name = ("dq", "dk", "dv")[i]
        assert_within(got, want[name], bound[name] + HALF_STEP, what + name)
    return grads


@pytest.mark.parametrize("do_size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("Sq,Skv", [(256, 8192), (4096, 512)])
@pytest.mark.parametrize("D", [64, 128])
def test_small_output_gradients(D, Sq, Skv, do_size):
    check(*make(1, 2, 2, Sq, Skv, D, do_size))


@pytest.mark.parametrize("do_size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("D,Sq,Skv", [(128, 256, 8192), (64, 4096, 512)])
def test_relative_errors_do_not_depend_on_the_size_of_the_output_gradients(D, Sq, Skv, do_size):
    """In the 2-norm, where the bounds above allow for thousands of errors of one sign: the roundings of P or dS, of out (in
    delta) and of the result are independent and each at most u = 2^-11 of what is rounded, so together they stay
    below 3 u of the result; and the result's own smallest half step."""
    q, k, v, do = make(1, 1, 1, Sq, Skv, D, do_size)
    grads = torch.autograd.grad(ops.cross_attention(q, k, v), (q, k, v), do)
    want, _ = cross_reference(q, k, v, None, None, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        off = float((got.double() - want[name]).norm())
        assert off <= 3 * 2.0 ** -11 * float(want[name].norm()) + HALF_STEP * math.sqrt(got.numel()), name


@pytest.mark.parametrize("asked", [(0,), (1, 2), (2,)])
def test_small_output_gradients_of_one_side(asked):
    """Without the query pass, the row statistics come from a kernel of their own."""
    args = make(2, 4, 2, 300, 2100, 64, 1e-4)
    whole = check(*args)
    alone = check(*args, asked=asked)
    assert all(torch.equal(a, whole[i]) for a, i in zip(alone, asked))


@pytest.mark.parametrize("asked", [(0, 1, 2), (1, 2)])
def test_many_key_heads(asked):
    """More key heads than the kernel of the row statistics has room for on the SM."""
    check(*make(300, 4, 4, 5, 7, 64, 1e-4), asked=asked)


@pytest.mark.parametrize("do_size", [1.0, 1e-4])
@pytest.mark.parametrize("size,kv_batch", [((3, 4, 2, 130, 700), None), ((3, 4, 2, 130, 700), 1), ((1, 3, 3, 200, 6000), None),
                                           ((1, 4, 2, 5000, 130), None), ((2, 3, 1, 1, 333), None)])
def test_masks_shared_heads_and_divided_units(size, kv_batch, do_size):
    q, k, v, do = make(*size, 128, do_size, kv_batch=kv_batch)
    check(q, k, v, do, what="no mask ")
    g = torch.Generator().manual_seed(1)
    holes = (torch.rand(size[0], size[4], generator=g) < 0.7).cuda()
    check(q, k, v, do, holes, "holes ")
    holes[0] = False
    check(q, k, v, do, holes, "one empty ")


@pytest.mark.parametrize("poison", [65504.0, math.inf, math.nan])
def test_masked_values_do_not_coarsen_the_others(poison):
    """What masked values hold, the type's largest number among it, takes no part in how dS is scaled."""
    q, k, v, do = make(2, 2, 2, 130, 700, 64, 1e-4)
    mask = torch.arange(700, device="cuda")[None] < torch.tensor([700, 300], device="cuda")[:, None]
    want = check(q, k, v, do, mask)
    with torch.no_grad():
        for t in (k, v):
            t.masked_fill_(~mask[:, None, :, None], poison)
    assert all(torch.equal(a, b) for a, b in zip(check(q, k, v, do, mask), want))
    # one set of states, kept by one batch entry and masked by the other
    q, k, v, do = make(2, 2, 2, 130, 700, 64, 1e-4, kv_batch=1)
    both = mask.clone()
    both[:, 600:] = False
    want = check(q, k, v, do, both)
    with torch.no_grad():
        for t in (k, v):
            t[:, :, 600:] = poison
    assert all(torch.equal(a, b) for a, b in zip(check(q, k, v, do, both), want))


def test_rows_and_heads_of_very_different_sizes():
    """Rows of dq have scales of their own; heads and batch entries too, for dk and dv."""
    q, k, v, do = make(2, 4, 2, 300, 1000, 64, 1.0)
    rows = torch.logspace(3, -4, 300, device="cuda")[None, None, :, None]
    check(q, k, v, (do.float() * rows).half(), asked=(0,))
    heads = torch.tensor([[1e-4, 1e-4, 1e2, 1e2], [1.0, 1.0, 1e-3, 1e-3]], device="cuda")[:, :, None, None]
    check(q, k, v, (do.float() * heads).half())
    some = do.clone()
    some[:, :, ::2] = 0.0
    some[0, 1] = 0.0
    check(q, k, v, some)
    check(q, k, v, torch.zeros_like(do))


def test_a_value_that_is_not_finite_stays_in_its_head():
    q, k, v, do = make(2, 4, 2, 130, 300, 64, 1e-4)
    want = check(q, k, v, do)
    bad = do.clone()
    bad[0, 0, 7, 3] = math.inf
    with torch.no_grad():
        v[1, 1, 5, 2] = math.inf
    dq, dk, dv = torch.autograd.grad(ops.cross_attention(q, k, v), (q, k, v), bad)
    assert not dq[0, 0, 7].isfinite().all() and not dk[0, 0].isfinite().any() and not dq[1, 2:].isfinite().any()
    keep = torch.ones(130, dtype=torch.bool)
    keep[7] = False
    assert torch.equal(dq[0, 1:], want[0][0, 1:]) and torch.equal(dq[1, :2], want[0][1, :2])
    assert torch.equal(dq[0, 0, keep], want[0][0, 0, keep])
    assert torch.equal(dk[0, 1], want[1][0, 1]) and torch.equal(dk[1, 0], want[1][1, 0])
    assert torch.equal(dv[0, 1], want[2][0, 1]) and torch.equal(dv[1, 0], want[2][1, 0])


def test_slopes_above_the_largest_f16_value():
    """dS passes 65504 where dq, dk and dv do not."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda s, size: (torch.randn(1, 2, s, 64, device="cuda", generator=g) * size).half()  # noqa: E731
    q, k, v, do = n(100, 0.05), n(4, 0.05), n(4, 8.0), n(100, 2000.0)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    want, _ = cross_reference(*leaves, None, None, do)
    weight = 0.25 * (do.double() @ v.detach().double().transpose(-1, -2)).abs().amax()
    assert weight.item() > 65504 and all(want[n].abs().max().item() < 65504 for n in ("dq", "dk", "dv"))
    check(*leaves, do)


@pytest.mark.parametrize("do_size", [1e-4, 1e-20])
def test_bfloat16_has_no_such_steps(do_size):
    q, k, v, do = make(1, 2, 2, 256, 8192, 64, do_size, dtype=torch.bfloat16)
    grads = torch.autograd.grad(ops.cross_attention(q, k, v), (q, k, v), do)
    want, bound = cross_reference(q, k, v, None, None, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, want[name], bound[name], name)


def test_captured_and_repeated():
    """The scales are found anew in every launch: a replay with other sizes of output gradients."""
    q, k, v, do = make(2, 4, 2, 130, 700, 128, 1e-4)
    leaves = (q, k, v)

    def step():
        return torch.autograd.grad(ops.cross_attention(*leaves), leaves, do)

    first = [t.clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, first))
    big = (do.float() * 4096).half()
    do.copy_(big)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
    check(q, k, v, do)
