"""ops.cross_attention against the definition in 64 bits: sizes around the tile edges, shared key
heads, broadcast states, masks, strides, gradients, streams and graphs. The bounds are derived in
block_ops_reference.py."""
import math

import pytest
import torch
import torch.utils.checkpoint

from block_ops_reference import assert_within, cross_reference
from paraattention_b200 import ops

pytestmark = pytest.mark.gpu


def make(B, Hq, Hkv, Sq, Skv, D, dtype=torch.bfloat16, seed=0, kv_batch=None, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(b, s, h):
        return torch.randn(b, s, h, D, device="cuda", generator=g).to(dtype).transpose(1, 2).requires_grad_(grad)

    kb = B if kv_batch is None else kv_batch
    return t(B, Sq, Hq), t(kb, Skv, Hkv), t(kb, Skv, Hkv), t(B, Sq, Hq).detach()


def check_forward(q, k, v, mask=None, scale=None, what=""):
    out, lse = ops.cross_attention(q, k, v, mask, scale=scale, return_lse=True)
    want, bound = cross_reference(q, k, v, mask, scale)
    assert_within(out, want["out"], bound["out"], what + "out")
    assert_within(lse, want["lse"], bound["lse"], what + "lse")
    return out, lse


def check_gradients(q, k, v, do, mask=None, scale=None, what=""):
    out = ops.cross_attention(q, k, v, mask, scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), do)
    want, bound = cross_reference(q, k, v, mask, scale, do)
    assert_within(out, want["out"], bound["out"], what + "out")
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, want[name], bound[name], what + name)
    return (out,) + grads


SIZES = [  # B, Hq, Hkv, Sq, Skv
    (1, 1, 1, 1, 1), (1, 2, 2, 1, 77), (2, 8, 2, 1, 333), (1, 16, 1, 1, 1000), (2, 4, 4, 16, 64), (1, 2, 1, 8, 65),
    (1, 1, 1, 17, 1), (1, 3, 3, 128, 128), (2, 2, 2, 129, 127), (1, 4, 2, 100, 129), (1, 6, 2, 257, 300), (2, 3, 1, 40, 63),
    (1, 2, 2, 300, 515), (1, 1, 1, 1024, 640),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", SIZES)
def test_forward_at_sizes_around_the_tile_edges(size, D, dtype):
    q, k, v, _ = make(*size, D, dtype)
    check_forward(q, k, v)


def masks(B, Skv, seed=0):
    g = torch.Generator().manual_seed(seed)
    tail = torch.arange(Skv)[None] < torch.randint(1, Skv + 1, (B, 1), generator=g)
    holes = torch.rand(B, Skv, generator=g) < 0.5
    front = torch.arange(Skv)[None] >= torch.randint(0, Skv, (B, 1), generator=g)
    empty = holes.clone()
    empty[0] = False
    return {"tail": tail, "holes": holes, "front": front, "empty": empty, "none": torch.zeros_like(holes),
            "all": torch.ones_like(holes), "last": torch.arange(Skv)[None].expand(B, -1) == Skv - 1,
            "one_row": holes[:1]}


@pytest.mark.parametrize("kind", ["tail", "holes", "front", "empty", "none", "all", "last", "one_row"])
@pytest.mark.parametrize("size,D", [((2, 4, 2, 1, 200), 128), ((3, 2, 2, 130, 333), 128), ((2, 2, 1, 70, 129), 64)])
def test_masks_and_rows_without_keys(size, D, kind):
    q, k, v, _ = make(*size, D)
    mask = masks(size[0], size[4])[kind].cuda()
    out, lse = check_forward(q, k, v, mask, what=kind + " ")
    nothing = ~mask.expand(size[0], -1).any(-1)
    if bool(nothing.any()):
        assert not out[nothing].any() and bool((lse[nothing] == -math.inf).all())
    # the 4-D form of attention masks is the same mask
    assert torch.equal(out, ops.cross_attention(q, k, v, mask[:, None, None, :]))


@pytest.mark.parametrize("size,D", [((2, 4, 2, 1, 200), 128), ((2, 2, 2, 130, 333), 128), ((2, 2, 1, 70, 129), 64)])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(size, D, poison):
    """Infinities and NaN in masked keys and values reach neither the output nor a gradient; the
    gradients of those places are zero."""
    q, k, v, do = make(*size, D)
    mask = masks(size[0], size[4])["empty"].cuda()
    hole = ~mask[:, None, :, None]
    kp, vp = (t.masked_fill(hole, poison).requires_grad_(True) for t in (k, v))
    q = q.detach().requires_grad_(True)
    got = check_gradients(q, kp, vp, do, mask)
    for g in got[2:]:
        assert not g.masked_select(hole).any()
    with torch.no_grad():
        check_forward(q, kp, vp, mask)


GRAD_SIZES = [  # B, Hq, Hkv, Sq, Skv
    (1, 1, 1, 1, 5), (2, 8, 2, 1, 77), (1, 2, 2, 16, 64), (1, 3, 3, 128, 128), (2, 2, 2, 129, 127), (1, 4, 2, 100, 129),
    (1, 6, 2, 257, 300), (1, 1, 1, 700, 1), (2, 3, 1, 40, 63), (1, 1, 1, 130, 1400),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", GRAD_SIZES)
def test_gradients_at_sizes_around_the_tile_edges(size, D, dtype):
    q, k, v, do = make(*size, D, dtype, grad=True)
    check_gradients(q, k, v, do)


@pytest.mark.parametrize("kind", ["tail", "holes", "front", "empty", "none", "last", "one_row"])
@pytest.mark.parametrize("size,D", [((3, 2, 2, 130, 333), 128), ((2, 4, 2, 70, 129), 64)])
def test_gradients_with_masks(size, D, kind):
    q, k, v, do = make(*size, D, grad=True)
    check_gradients(q, k, v, do, masks(size[0], size[4])[kind].cuda(), what=kind + " ")


@pytest.mark.parametrize("kind", [None, "tail", "empty"])
@pytest.mark.parametrize("size,D", [((3, 4, 2, 70, 200), 128), ((4, 2, 2, 1, 130), 64), ((3, 2, 1, 300, 257), 128)])
def test_one_set_of_states_for_the_whole_batch(size, D, kind):
    """Keys and values of batch size 1: their gradients are the sums over the batch."""
    q, k, v, do = make(*size, D, kv_batch=1, grad=True)
    mask = None if kind is None else masks(size[0], size[4])[kind].cuda()
    check_gradients(q, k, v, do, mask)
    with torch.no_grad():
        a, _ = check_forward(q, k, v, mask)
        # the same states expanded over the batch
        b = ops.cross_attention(q, k.expand(size[0], -1, -1, -1), v.expand(size[0], -1, -1, -1), mask)
        assert torch.equal(a, b)
    # ... whose gradients PyTorch sums
    ke, ve = k.expand(size[0], -1, -1, -1), v.expand(size[0], -1, -1, -1)
    grads = torch.autograd.grad(ops.cross_attention(q, ke, ve, mask), (k, v), do)
    want, bound = cross_reference(q, k, v, mask, None, do)
    for name, got in zip(("dk", "dv"), grads):
        # (each batch entry's gradient is rounded, and so is PyTorch's sum of them)
        extra = 2.0 ** -7 * cross_abs(q, k, v, mask, do)[name]
        assert_within(got, want[name], bound[name] + extra, name)


def cross_abs(q, k, v, mask, do):
    """Sums over the batch of the batch entries' absolute gradients."""
    B = q.shape[0]
    vals, _ = cross_reference(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), mask, None, do)
    return {n: vals[n].abs().sum(0, keepdim=True) for n in ("dk", "dv")}


@pytest.mark.parametrize("D", [64, 128])
def test_long_keys_are_divided_over_the_sms(D):
    """Few rows against many keys: several CTAs share a unit and their partial results are joined."""
    q, k, v, do = make(1, 3, 3, 200, 6000, D, grad=True)
    first = check_gradients(q, k, v, do)
    again = check_gradients(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # fixed order of the sums
    mask = (torch.arange(6000, device="cuda") < 3001)[None]
    check_gradients(q, k, v, do, mask)


def test_long_queries_are_divided_over_the_sms():
    """Few key tiles against many rows (the key pass of the backward kernel is split)."""
    q, k, v, do = make(1, 4, 2, 5000, 130, 128, grad=True)
    first = check_gradients(q, k, v, do)
    again = check_gradients(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_more_units_than_ctas():
    """Several units per CTA, with different numbers of key tiles (masks) and empty ones among them."""
    q, k, v, do = make(6, 16, 16, 300, 260, 64, grad=True)
    mask = torch.arange(260)[None] < torch.tensor([260, 0, 1, 128, 129, 40])[:, None]
    check_gradients(q, k, v, do, mask.cuda())
    check_gradients(q, k, v, do)


@pytest.mark.parametrize("Sq", [1, 40])
def test_strides_and_alignment(Sq):
    """Packed projections, [B, H, S, D] memory, transposed heads, misaligned bases: same values."""
    B, H, Skv, D = 2, 4, 100, 64
    q, k, v, _ = make(B, H, H, Sq, Skv, D)
    want = ops.cross_attention(q, k, v)
    packed = torch.cat([k.transpose(1, 2).flatten(2), v.transpose(1, 2).flatten(2)], dim=-1)
    kp, vp = (t.unflatten(-1, (H, D)).transpose(1, 2) for t in packed.chunk(2, dim=-1))
    assert torch.equal(want, ops.cross_attention(q, kp, vp))
    assert torch.equal(want, ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous()))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(B, H, Sq, D).copy_(q)
    assert torch.equal(want, ops.cross_attention(odd, k, v))
    wide = torch.zeros(B, H, Skv, D + 4, dtype=q.dtype, device="cuda")  # rows of 136 bytes: not 16-byte steps
    wide[..., :D] = k
    assert torch.equal(want, ops.cross_attention(q, wide[..., :D], v))
    column = k.transpose(-1, -2).contiguous().transpose(-1, -2)  # head_dim not contiguous
    assert torch.equal(want, ops.cross_attention(q, column, v))
    mask = torch.rand(Skv, B, device="cuda") < 0.7  # [B, Skv] as a transposed view
    assert torch.equal(ops.cross_attention(q, k, v, mask.t()), ops.cross_attention(q, k, v, mask.t().contiguous()))


def test_gradients_of_strided_inputs_and_output_gradients():
    B, H, Sq, Skv, D = 2, 4, 130, 100, 64
    q, k, v, do = make(B, H, H, Sq, Skv, D, grad=True)
    want = check_gradients(q, k, v, do)
    packed = torch.cat([k.transpose(1, 2).flatten(2), v.transpose(1, 2).flatten(2)], dim=-1).detach().requires_grad_(True)
    kp, vp = (t.unflatten(-1, (H, D)).transpose(1, 2) for t in packed.chunk(2, dim=-1))
    out = ops.cross_attention(q, kp, vp)
    dq, dpacked = torch.autograd.grad(out, (q, packed), do.contiguous())
    dk, dv = (t.unflatten(-1, (H, D)).transpose(1, 2) for t in dpacked.chunk(2, dim=-1))
    assert torch.equal(dq, want[1]) and torch.equal(dk, want[2]) and torch.equal(dv, want[3])
    # a broadcast output gradient (sum) is a zero-stride tensor
    ones = torch.ones_like(do)
    a = torch.autograd.grad(ops.cross_attention(q, k, v).sum(), (q, k, v))
    b = torch.autograd.grad(ops.cross_attention(q, k, v), (q, k, v), ones)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradients_only_where_they_are_asked_for():
    q, k, v, do = make(1, 2, 2, 130, 100, 64)
    out = ops.cross_attention(q, k, v)
    assert not out.requires_grad
    k.requires_grad_(True)
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    assert out.requires_grad and not lse.requires_grad
    out.backward(do)
    want, bound = cross_reference(q, k, v, None, None, do)
    assert_within(k.grad, want["dk"], bound["dk"], "dk")
    assert q.grad is None and v.grad is None
    with torch.no_grad():
        assert not ops.cross_attention(q, k, v).requires_grad


def test_gradients_against_differences():
    """The directional derivative of a smooth scalar of the output, in f16 with inputs on a coarse grid so
    that the shifted inputs are exact; central differences of the 64-bit definition."""
    q, k, v, _ = make(1, 2, 1, 20, 70, 64, torch.float16)
    q, k, v = ((t * 8).round() / 8 for t in (q, k, v))
    weight = torch.randn(1, 2, 20, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, weight)
    h = 2.0 ** -7
    _, bound = cross_reference(q, k, v, None, None, weight)
    for i, (name, g) in enumerate(zip(("dq", "dk", "dv"), grads)):
        step = torch.zeros(leaves[i].shape, dtype=torch.float64, device="cuda")
        step.view(-1)[::37] = 1.0

        def f(sign):
            args = [t.detach().double() for t in leaves]
            args[i] = args[i] + sign * h * step
            vals, _ = cross_reference(*(a for a in args))
            return float((vals["out"] * weight.double()).sum())

        slope = (f(1) - f(-1)) / (2 * h)
        got = float((g.double() * step).sum())
        room = float((bound[name] * step).sum()) + 1e-3 * abs(slope) + 1e-3  # (h^2 of the third derivative)
        assert abs(got - slope) <= room, f"{name}: {got} against {slope} +- {room}"


def test_scale_and_large_logits():
    q, k, v, do = make(1, 2, 2, 150, 200, 128, grad=True)
    check_gradients(q, k, v, do, scale=0.5)  # logits of standard deviation 5.7: near one-hot rows
    q1, k1, v1, _ = make(1, 2, 2, 1, 200, 128)
    check_forward(q1, k1, v1, scale=0.5)
    # rows whose logits are all far from zero
    shift = torch.full_like(k.detach(), 2.0)
    check_forward(q.detach(), k.detach() + shift, v.detach(), scale=0.5)


def test_lengths_of_zero():
    q, k, v, do = make(2, 2, 2, 5, 7, 64, grad=True)
    out, lse = ops.cross_attention(q, k[:, :, :0], v[:, :, :0], return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    grads = torch.autograd.grad(out, (q, k, v), do)
    assert not any(bool(g.any()) for g in grads)
    assert ops.cross_attention(q[:, :, :0], k, v).shape == (2, 2, 0, 64)
    assert ops.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 2, 5, 64)


def test_other_streams_and_graphs():
    q, k, v, do = make(2, 4, 2, 130, 333, 128, grad=True)
    mask = masks(2, 333)["tail"].cuda()

    def step():
        out = ops.cross_attention(q, k, v, mask)
        return (out,) + torch.autograd.grad(out, (q, k, v), do)

    want = [t.detach().clone() for t in step()]
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
    with torch.no_grad():  # other inputs in the same memory
        for t in (q, k, v):
            t.copy_(t.roll(1, dims=2))
        mask.copy_(masks(2, 333, seed=5)["holes"])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in got]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # single tokens too
    q1, k1, v1, _ = make(2, 4, 2, 1, 333, 128)
    ops.cross_attention(q1, k1, v1, mask)
    graph1 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph1):
        out1 = ops.cross_attention(q1, k1, v1, mask)
    q1.copy_(q1.flip(1))
    graph1.replay()
    assert torch.equal(out1, ops.cross_attention(q1, k1, v1, mask))


def test_calls_at_once_on_two_streams():
    """Two backward passes in flight have workspaces of their own."""
    sets = [make(1, 3, 3, 200, 6000, 128, seed=s, grad=True) for s in (1, 2)]

    def step(q, k, v, do):
        out = ops.cross_attention(q, k, v)
        return (out,) + torch.autograd.grad(out, (q, k, v), do)

    want = [[t.detach().clone() for t in step(*s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(step(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("Sq,Skv", [(1, 100), (5, 333), (200, 300), (130, 4000)])
def test_infinite_logits_and_nan_in_places_that_take_part(Sq, Skv):
    """A key whose logits are -inf has weight zero, also where a whole run of keys is like that; NaN stays in the
    rows that see it (the last size is divided over several CTAs)."""
    q, k, v, _ = make(1, 2, 2, Sq, Skv, 64)
    q[..., 0] = 1.0
    k[:, :, :90, 0] = -math.inf
    keep = torch.arange(Skv, device="cuda")[None] >= 90
    kept = k.clone()
    kept[:, :, :90, 0] = 0.0
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    want, bound = cross_reference(q, kept, v, keep, None)
    assert_within(out, want["out"], bound["out"], "out")
    assert_within(lse, want["lse"], bound["lse"], "lse")

    q, k, v, do = make(1, 2, 2, Sq, Skv, 64, grad=True)
    clean, clean_lse = ops.cross_attention(q, k, v, return_lse=True)
    with torch.no_grad():
        q[0, 0, Sq - 1, 3] = math.nan
        k[0, 1, Skv - 1, 5] = math.nan
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    assert out[0, 0, Sq - 1].isnan().all() and lse[0, 0, Sq - 1].isnan() and out[0, 1].isnan().all() and lse[0, 1].isnan().all()
    assert torch.equal(out[0, 0, :Sq - 1], clean[0, 0, :Sq - 1]) and torch.equal(lse[0, 0, :Sq - 1], clean_lse[0, 0, :Sq - 1])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert dq[0, 0, Sq - 1].isnan().all() and dk[0, 0].isnan().all() and dv[0, 0].isnan().all() and dq[0, 1].isnan().all()
    assert not dq[0, 0, :Sq - 1].isnan().any()


@pytest.mark.parametrize("asked", [(0,), (1,), (2,), (0, 2), (1, 2)])
@pytest.mark.parametrize("Sq", [1, 300])
def test_gradients_alone_equal_those_of_the_whole_call(Sq, asked):
    q, k, v, do = make(2, 4, 2, Sq, 200, 128, grad=True)
    whole = check_gradients(q, k, v, do)[1:]
    xs = [x if i in asked else x.detach() for i, x in enumerate((q, k, v))]
    got = torch.autograd.grad(ops.cross_attention(*xs), [xs[i] for i in asked], do)
    assert all(torch.equal(a, whole[i]) for a, i in zip(got, asked))


def test_tensors_saved_elsewhere_between_forward_and_backward():
    q, k, v, do = make(2, 4, 2, 300, 200, 64, grad=True)
    mask = masks(2, 200)["holes"].cuda()
    want = check_gradients(q, k, v, do, mask)[1:]
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        out = ops.cross_attention(q, k, v, mask)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), do), want))
    out = torch.utils.checkpoint.checkpoint(lambda *a: ops.cross_attention(*a), q, k, v, mask, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), do), want))


@pytest.mark.parametrize("Sq", [3, 200])
def test_rows_more_than_four_gigabytes_apart(Sq):
    """Keys, values and queries as views with a row step of 2 MB over a buffer of 5 GB: offsets pass 32 bits."""
    B, H, Skv, D, step = 1, 1, 2400, 64, 1 << 20
    big = torch.empty(Skv * step, dtype=torch.bfloat16, device="cuda")
    q, k, v, do = make(B, H, H, Sq, Skv, D)
    far = lambda at, rows: big.as_strided((B, H, rows, D), (0, 0, step, 1), at)  # noqa: E731
    kf, vf, qf = far(0, Skv), far(64, Skv), far(128, Sq)
    for f, x in ((kf, k), (vf, v), (qf, q)):
        f.copy_(x)
    leaves = [t.requires_grad_(True) for t in (qf, kf, vf)]
    want = check_gradients(*leaves, do)
    near = [t.detach().contiguous().requires_grad_(True) for t in leaves]
    out = ops.cross_attention(*near)
    assert torch.equal(out, want[0])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, near, do), want[1:]))
    assert torch.equal(ops.cross_attention(*(t.detach() for t in leaves)), want[0])


@pytest.mark.parametrize("size", [(1, 200, 1, 1, 40), (300, 2, 2, 1, 9), (40, 3, 3, 18, 5), (2, 16, 1, 1, 70), (2, 17, 1, 1, 70)])
def test_many_units_of_few_rows(size):
    """Many heads or sequences with hardly any rows: both sides of the limit of 16 rows per key head."""
    q, k, v, do = make(*size, 64, grad=True)
    check_gradients(q, k, v, do)
    with torch.no_grad():
        check_forward(q, k, v)


def test_what_lies_behind_the_tensors_is_left_alone():
    """Rows of a larger buffer behind the last key and query are neither read nor written."""
    B, H, Sq, Skv, D = 1, 2, 37, 45, 64
    for rows in (1, Sq):
        big_q = torch.full((B, 64, H, D), math.nan, dtype=torch.bfloat16, device="cuda")
        big_k, big_v = big_q.clone(), big_q.clone()
        q, k, v, do = make(B, H, H, rows, Skv, D)
        big_q[:, :rows], big_k[:, :Skv], big_v[:, :Skv] = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
        views = [big_q[:, :rows].transpose(1, 2), big_k[:, :Skv].transpose(1, 2), big_v[:, :Skv].transpose(1, 2)]
        leaves = [t.requires_grad_(True) for t in views]
        check_gradients(*leaves, do)
        assert bool(big_q[:, rows:].isnan().all()) and bool(big_k[:, Skv:].isnan().all())


def test_a_reported_timeout_stops_later_calls_until_it_is_reset():
    """The device's status word (set here by hand, as a wait that gave up would): tile kernels return at once and
    leave their outputs alone; the host's word makes the next call raise; both are cleared by a reset."""
    from paraattention_b200 import _lib as L
    from paraattention_b200 import _status

    q, k, v, do = make(1, 2, 2, 300, 200, 64, grad=True)
    want = check_gradients(q, k, v, do)
    recorded = ops.cross_attention(q, k, v)
    mirror = _status.single_gpu_status(q.device)
    try:
        mirror.word.fill_(L.PA_DEV_TIMEOUT_PIPE)
        out, lse = ops.cross_attention(q.detach(), k.detach(), v.detach(), return_lse=True)
        torch.cuda.synchronize()
        mirror.host.fill_(L.PA_DEV_TIMEOUT_PIPE)
        with pytest.raises(L.PaError) as e:
            ops.cross_attention(q.detach(), k.detach(), v.detach())
        assert e.value.code == L.PA_ETIMEDOUT
        with pytest.raises(RuntimeError, match="gave up waiting"):
            torch.autograd.grad(recorded, (q, k, v), do)
    finally:
        mirror.reset()
    again = check_gradients(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_first_call_inside_a_capture():
    """Without a status word made yet, a captured call does without one."""
    from paraattention_b200 import _status

    q, k, v, _ = make(1, 2, 2, 200, 300, 64)
    want = ops.cross_attention(q, k, v)
    kept = dict(_status._single)
    _status._single.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.cross_attention(q, k, v)
        assert not _status._single
    finally:
        _status._single.update(kept)
    graph.replay()
    assert torch.equal(out, want)


def test_refusals():
    q, k, v, _ = make(2, 4, 2, 5, 7, 64)
    with pytest.raises(NotImplementedError, match="bfloat16 and float16"):
        ops.cross_attention(q.float(), k.float(), v.float())
    with pytest.raises(NotImplementedError, match="head_dim 32"):
        ops.cross_attention(q[..., :32], k[..., :32], v[..., :32])
    with pytest.raises(AssertionError, match="multiple"):
        ops.cross_attention(q[:, :3], k, v)
    with pytest.raises(AssertionError, match="batch of key"):
        ops.cross_attention(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1))
    with pytest.raises(AssertionError, match="boolean"):
        ops.cross_attention(q, k, v, torch.ones(2, 7, device="cuda"))
    with pytest.raises(NotImplementedError, match="key-padding"):
        ops.cross_attention(q, k, v, torch.ones(2, 1, 5, 7, dtype=torch.bool, device="cuda"))
    with pytest.raises(AssertionError, match="device"):
        ops.cross_attention(q, k, v, torch.ones(2, 7, dtype=torch.bool))
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            ops.cross_attention(q, k, v, scale=scale)
    q = q.detach().requires_grad_(True)
    g, = torch.autograd.grad(ops.cross_attention(q, k, v).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):  # first derivatives only
        torch.autograd.grad(g.float().sum(), q)
