"""Cross attention and the q/k norm with rotation as a transformer block uses them: together, through
the mode, and inside the shape-only transformers, forward and backward."""
import math

import pytest
import torch
import torch.nn.functional as F

import paraattention_b200 as pa
from block_ops_reference import unit
from paraattention_b200 import config, ops

pytestmark = pytest.mark.gpu


def _rel(got, want):
    got, want = got.double(), want.double()
    return float((got - want).norm() / want.norm().clamp_min(1e-300))


def _turn64(x, cos, sin):
    o = torch.empty_like(x)
    o[..., ::2] = x[..., ::2] * cos[:, ::2] - x[..., 1::2] * sin[:, ::2]
    o[..., 1::2] = x[..., 1::2] * cos[:, 1::2] + x[..., ::2] * sin[:, 1::2]
    return o


@pytest.mark.parametrize("masked", [False, True])
def test_norm_rotation_and_attention_together(masked):
    """Normalised, rotated queries against normalised prompt keys, as a video block's attention: the
    gradients of everything that goes in, against the same chain in 64 bits under PyTorch's autograd. On the
    way to a result lie at most seven roundings (y, P, out, delta, dS, dq, dx), whose relative errors of at
    most u each add up to 8 u in the 2-norm (their products are smaller still)."""
    B, H, Hk, S, T, D = 2, 4, 2, 300, 150, 128
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(7)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    raw = {"q": n(B, S, H, D), "k": n(B, T, Hk, D), "v": n(B, T, Hk, D)}
    raw = {k: v.to(dt).transpose(1, 2) for k, v in raw.items()}
    raw |= {w: (1 + 0.2 * n(D)).to(dt) for w in ("wq", "wk")}
    ang = n(S, D // 2).repeat_interleave(2, dim=-1)
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    do = n(B, S, H, D).to(dt).transpose(1, 2)
    mask = (torch.arange(T, device="cuda")[None] < torch.tensor([T, 61], device="cuda")[:, None]) if masked else None

    x = {k: v.clone().requires_grad_(True) for k, v in raw.items()}
    qn, _ = ops.qk_norm_rotary(x["q"], None, x["wq"], None, (cos, sin))
    kn, _ = ops.qk_norm_rotary(x["k"], None, x["wk"])
    out = ops.cross_attention(qn, kn, x["v"], mask)
    out.backward(do)

    y = {k: v.double().requires_grad_(True) for k, v in raw.items()}
    norm = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    q64 = _turn64(norm(y["q"], y["wq"]), cos.double(), sin.double())
    k64, v64 = (t.repeat_interleave(H // Hk, dim=1) for t in (norm(y["k"], y["wk"]), y["v"]))
    z = torch.einsum("bhmd,bhnd->bhmn", q64, k64) / math.sqrt(D)
    if masked:
        z = z.masked_fill(~mask[:, None, None, :], -math.inf)
    want = torch.einsum("bhmn,bhnd->bhmd", torch.softmax(z, -1), v64)
    want.backward(do.double())
    bound = 8 * unit(dt)
    assert _rel(out, want) <= bound
    for name in raw:
        assert _rel(x[name].grad, y[name].grad) <= bound, name


def _tiny_wan():
    from paraattention_b200.shape_models_video import WanShapedTransformer3DModel

    torch.manual_seed(0)
    return WanShapedTransformer3DModel(dim=256, num_layers=2, ffn_dim=512, text_dim=64).cuda().bfloat16()


def _wan_step(model):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, 16, 2, 16, 16, device="cuda", generator=g).bfloat16()
    enc = torch.randn(1, 33, 64, device="cuda", generator=g).bfloat16()
    target = torch.randn(1, 16, 2, 16, 16, device="cuda", generator=g)
    out = model(x, torch.tensor([500.0], device="cuda"), enc).sample
    (out.float() - target).square().mean().backward()
    return out


def test_a_transformer_trains_through_the_kernels():
    """A Wan-shaped transformer step with the differentiable operators: every parameter gets a finite
    gradient, and the gradients agree with those of the chain of tensor operations under PyTorch's own attention
    (both in bf16: two computations of the same function with some twenty roundings on each side between a
    parameter and the loss, so 40 u of the gradient's size)."""
    kernels, eager = _tiny_wan(), _tiny_wan()
    with config.patch({"attention.differentiable": True}), pa.CrossAttnMode(same_length=True):
        out = _wan_step(kernels)
    with config.patch({"attention.fuse_qkv_prepare": False}):
        want = _wan_step(eager)
    assert _rel(out, want) <= 40 * unit(torch.bfloat16)
    for (name, p), (_, e) in zip(kernels.named_parameters(), eager.named_parameters()):
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
        if e.grad is not None and float(e.grad.float().norm()) > 0:
            assert _rel(p.grad, e.grad) <= 40 * unit(torch.bfloat16), name


def test_partial_rotation_of_joint_streams_with_gradients():
    """Video then text, rotation on the video rows only: the differentiable preparation against the eager chain."""
    from paraattention_b200.shape_models import _joint_qkv

    g = torch.Generator(device="cuda").manual_seed(0)
    H, D, n_img, n_txt = 2, 128, 70, 40

    def stream(rows):
        p = [torch.randn(1, rows, H * D, device="cuda", generator=g).bfloat16().requires_grad_(True) for _ in range(3)]
        w = [(1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16().requires_grad_(True) for _ in range(2)]
        return (*p, *w)

    streams = [stream(n_img), stream(n_txt)]
    ang = torch.rand(n_img, D // 2, device="cuda", generator=g).repeat_interleave(2, dim=-1) * 6.28
    rotary = (ang.cos().contiguous(), ang.sin().contiguous())
    leaves = [t for s in streams for t in s]
    do = [torch.randn(1, H, n_img + n_txt, D, device="cuda", generator=g).bfloat16() for _ in range(3)]
    for rows in ((0, n_img), None):
        tab = rotary if rows else tuple(torch.cat([t, t[:n_txt]]) for t in rotary)
        with config.patch({"attention.differentiable": True}):
            got = _joint_qkv(streams, tab, rotary_rows=rows)
        with config.patch({"attention.fuse_qkv_prepare": False}):
            want = _joint_qkv(streams, tab, rotary_rows=rows)
        a, b = (torch.autograd.grad(o, leaves, do) for o in (got, want))
        # (one rounding against the chain's three and their gradients')
        for x, y in zip(list(got) + list(a), list(want) + list(b)):
            assert _rel(x, y) <= 6 * unit(torch.bfloat16)
        with torch.no_grad(), config.patch({"attention.differentiable": True}):
            plain = _joint_qkv(streams, tab, rotary_rows=rows)  # nothing recorded: the fused kernel
        with torch.no_grad():
            assert all(torch.equal(x, y) for x, y in zip(plain, _joint_qkv(streams, tab, rotary_rows=rows)))


def test_mode_routes_cross_attention_with_masks_and_shared_heads():
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(2, 8, 100, 64, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(2, 2, 30, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    mask = torch.rand(2, 1, 1, 30, device="cuda", generator=g) < 0.6
    with pa.CrossAttnMode():
        got = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=0.2, enable_gqa=True)
    assert torch.equal(got, ops.cross_attention(q, k, v, mask, scale=0.2))
