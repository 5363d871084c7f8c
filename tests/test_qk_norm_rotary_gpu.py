"""ops.qk_norm_rotary (per-head norm of queries and keys with the position rotation, forward and
backward) against the definition in 64 bits; bounds in block_ops_reference.py."""
import math

import pytest
import torch

from block_ops_reference import assert_within, norm_reference
from paraattention_b200 import ops

pytestmark = pytest.mark.gpu


def make(B, Hq, Hk, S, D, dtype, interleaved=True, seed=0, grad=False, rows=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q = (2 * n(B, S, Hq, D)).to(dtype).transpose(1, 2)
    k = (2 * n(B, S, Hk, D)).to(dtype).transpose(1, 2)
    wq, wk = ((1 + 0.2 * n(D)).to(dtype) for _ in range(2))
    # (tables of any values: the two elements of a pair have angles of their own)
    ang = n(rows or S, D) * 3
    rotary = (ang.cos().contiguous(), ang.sin().contiguous())
    dq, dk = n(B, S, Hq, D).to(dtype).transpose(1, 2), n(B, S, Hk, D).to(dtype).transpose(1, 2)
    for t in (q, k, wq, wk):
        t.requires_grad_(grad)
    return q, k, wq, wk, rotary, dq, dk


def check(q, k, wq, wk, rotary, interleaved, dq=None, dk=None, eps=1e-6, row_offset=0):
    yq, yk = ops.qk_norm_rotary(q, k, wq, wk, rotary, eps=eps, interleaved=interleaved, row_offset=row_offset)
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    grads = dict(zip((id(t) for t in leaves), torch.autograd.grad((yq, yk), leaves, (dq, dk)))) if dq is not None else {}
    for name, x, w, y, dy in (("q", q, wq, yq, dq), ("k", k, wk, yk, dk)):
        want, bound = norm_reference(x, w, rotary, interleaved, eps, row_offset, dy)
        assert_within(y, want["y"], bound["y"], name)
        assert y.transpose(1, 2).is_contiguous()
        if dy is not None:
            assert_within(grads[id(x)], want["dx"], bound["dx"], "d" + name)
            if w is not None:
                assert_within(grads[id(w)], want["dw"], bound["dw"], "dw" + name)


SIZES = [(1, 1, 1, 1), (2, 4, 4, 7), (1, 24, 24, 130), (8, 32, 8, 1), (2, 3, 1, 65), (1, 40, 5, 333), (3, 1, 7, 20)]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hq,Hk,S", SIZES)
def test_values_and_gradients(B, Hq, Hk, S, D, dtype, interleaved):
    q, k, wq, wk, rotary, dq, dk = make(B, Hq, Hk, S, D, dtype, grad=True)
    check(q, k, wq, wk, rotary, interleaved, dq, dk)
    with torch.no_grad():
        check(q, k, wq, wk, rotary, interleaved)


@pytest.mark.parametrize("interleaved", [True, False])
def test_parts_may_be_missing(interleaved):
    """No rotation, no weights, no k; a table offset; another eps."""
    q, k, wq, wk, rotary, dq, dk = make(2, 4, 2, 33, 64, torch.bfloat16, grad=True, rows=50)
    check(q, k, wq, wk, None, interleaved, dq, dk)
    check(q, k, None, None, rotary, interleaved, dq, dk)
    check(q, k, wq, None, rotary, interleaved, dq, dk, row_offset=17)
    check(q, k, wq, wk, rotary, interleaved, dq, dk, eps=0.5, row_offset=3)
    y, none = ops.qk_norm_rotary(q, None, wq, None, rotary, interleaved=interleaved)
    assert none is None
    want, bound = norm_reference(q, wq, rotary, interleaved, 1e-6, 0, dq)
    g, gw = torch.autograd.grad(y, (q, wq), dq)
    assert_within(y, want["y"], bound["y"], "q")
    assert_within(g, want["dx"], bound["dx"], "dq")
    assert_within(gw, want["dw"], bound["dw"], "dwq")
    same, _ = ops.qk_norm_rotary(q.detach())
    assert torch.equal(same, q)


def test_only_the_gradients_asked_for():
    q, k, wq, wk, rotary, dq, dk = make(1, 4, 2, 40, 64, torch.bfloat16, grad=False)
    full = make(1, 4, 2, 40, 64, torch.bfloat16, grad=True)
    want = torch.autograd.grad(ops.qk_norm_rotary(*full[:4], rotary), full[:4], (dq, dk))
    args = [q, k, wq, wk]
    for asked in ([0], [1], [2], [3], [0, 3], [1, 2]):
        leaves = [t.detach().requires_grad_(i in asked) for i, t in enumerate(args)]
        yq, yk = ops.qk_norm_rotary(*leaves, rotary)
        got = torch.autograd.grad((yq, yk), [leaves[i] for i in asked], (dq, dk), allow_unused=True)
        for i, g in zip(asked, got):
            assert torch.equal(g, want[i]), f"input {i}"
    # one output unused: its gradient is zero
    leaves = [t.detach().requires_grad_(True) for t in args]
    yq, yk = ops.qk_norm_rotary(*leaves, rotary)
    got = torch.autograd.grad(yq, leaves, dq)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and not got[1].any() and not got[3].any()
    assert not ops.qk_norm_rotary(*args, rotary)[0].requires_grad


def test_strides_alignment_and_zero_rows():
    B, H, S, D = 2, 4, 33, 64
    q, k, wq, wk, rotary, _, _ = make(B, H, H, S, D, torch.bfloat16)
    want = ops.qk_norm_rotary(q, k, wq, wk, rotary)
    packed = torch.cat([t.transpose(1, 2).flatten(2) for t in (q, k)], dim=-1)
    qp, kp = (t.unflatten(-1, (H, D)).transpose(1, 2) for t in packed.chunk(2, dim=-1))
    for a, b in ((qp, kp), (q.contiguous(), k.contiguous()),
                 (torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(B, H, S, D).copy_(q), k),
                 (q.transpose(-1, -2).contiguous().transpose(-1, -2), k)):
        got = ops.qk_norm_rotary(a, b, wq, wk, rotary)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w_odd = torch.empty(D + 1, dtype=wq.dtype, device="cuda")[1:].copy_(wq)
    tab = [torch.empty(t.numel() + 1, device="cuda")[1:].view_as(t).copy_(t) for t in rotary]
    got = ops.qk_norm_rotary(q, k, w_odd, wk, tuple(tab))
    assert torch.equal(got[0], want[0])
    # a row of zeros has no direction: the norm gives zero, and a finite gradient
    z = torch.zeros(1, 2, 3, D, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y, _ = ops.qk_norm_rotary(z, None, wq, None, None)
    g, = torch.autograd.grad(y, z, torch.ones_like(y))
    assert not y.any() and bool(g.isfinite().all())
    assert ops.qk_norm_rotary(q[:, :, :0], k[:, :, :0], wq, wk, rotary)[0].shape == (B, H, 0, D)
    none, some = ops.qk_norm_rotary(q[:, :0], k, wq, wk, rotary)
    assert none.shape == (B, 0, S, D) and torch.equal(some, want[1])
    leaves = [t.detach().requires_grad_(True) for t in (q[:, :0], k, wq, wk)]
    y = ops.qk_norm_rotary(*leaves, rotary)
    grads = torch.autograd.grad(y, leaves, [torch.ones_like(t) for t in y])
    assert grads[0].numel() == 0 and not grads[2].any() and bool(grads[3].any())


def test_rows_more_than_four_gigabytes_apart():
    step, S, D = 1 << 20, 2400, 64
    big = torch.empty(S * step, dtype=torch.bfloat16, device="cuda")
    q, _, wq, _, rotary, dq, _ = make(1, 1, 1, S, D, torch.bfloat16)
    far = big.as_strided((1, 1, S, D), (0, 0, step, 1)).copy_(q).requires_grad_(True)
    near = q.detach().requires_grad_(True)
    a, b = (ops.qk_norm_rotary(t, None, wq, None, rotary)[0] for t in (far, near))
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, far, dq)[0], torch.autograd.grad(b, near, dq)[0])


def test_repeats_streams_and_graphs_give_the_same_bits():
    q, k, wq, wk, rotary, dq, dk = make(2, 8, 2, 1500, 128, torch.bfloat16, grad=True)
    leaves = (q, k, wq, wk)

    def step():
        y = ops.qk_norm_rotary(*leaves, rotary)
        return tuple(y) + torch.autograd.grad(y, leaves, (dq, dk))

    want = [t.detach().clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        q.copy_(q.flip(2))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals():
    q, k, wq, wk, rotary, _, _ = make(2, 4, 2, 9, 64, torch.bfloat16)
    with pytest.raises(NotImplementedError, match="bfloat16 and float16"):
        ops.qk_norm_rotary(q.float(), k.float())
    with pytest.raises(NotImplementedError, match="head_dim"):
        ops.qk_norm_rotary(q[..., :32], k[..., :32])
    with pytest.raises(AssertionError, match="agree"):
        ops.qk_norm_rotary(q, k[:, :, :5])
    with pytest.raises(AssertionError, match="weights"):
        ops.qk_norm_rotary(q, k, wq.float(), wk)
    with pytest.raises(AssertionError, match="tables end"):
        ops.qk_norm_rotary(q, k, wq, wk, rotary, row_offset=1)
    with pytest.raises(AssertionError, match="fp32"):
        ops.qk_norm_rotary(q, k, wq, wk, tuple(t.bfloat16() for t in rotary))
    with pytest.raises(AssertionError, match="k_weight"):
        ops.qk_norm_rotary(q, None, wq, wk)
    with pytest.raises(NotImplementedError, match="gradient of cos"):
        ops.qk_norm_rotary(q, k, wq, wk, (rotary[0].clone().requires_grad_(True), rotary[1]))
    for eps in (-1.0, math.nan):
        with pytest.raises(ValueError, match="eps"):
            ops.qk_norm_rotary(q, k, eps=eps)
