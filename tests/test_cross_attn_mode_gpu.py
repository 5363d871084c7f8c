"""pa.CrossAttnMode hands on the calls that ops.cross_attention does not compute."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

import paraattention_b200 as pa
from paraattention_b200 import ops

pytestmark = pytest.mark.gpu


def make(B=2, H=2, Sq=200, Skv=150, D=64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, s, H, D, device="cuda", generator=g).bfloat16().transpose(1, 2) for s in (Sq, Skv, Skv)]


def _sdpa(q, k, v, **kw):
    return F.scaled_dot_product_attention(q, k, v, **kw)


def test_the_mode_hands_on_what_the_operator_does_not_compute():
    """Calls with keys of another length that PyTorch serves and this operator does not are PyTorch's."""
    q, k, v = make(D=64)
    B, H, Sq, Skv = 2, 2, 200, 150
    g = torch.Generator(device="cuda").manual_seed(5)
    additive = torch.randn(B, 1, 1, Skv, device="cuda", generator=g).bfloat16()
    per_query = torch.rand(B, 1, Sq, Skv, device="cuda", generator=g) < 0.7
    wide = [torch.cat([t, t], dim=-1)[..., :96] for t in (q, k, v)]
    calls = [((q, k, v), {"attn_mask": additive}), ((q, k, v), {"attn_mask": per_query}),
             (tuple(t.float() for t in (q, k, v)), {}), (tuple(wide), {}), ((q, k, v), {"is_causal": True}),
             (tuple(t[:, 0] for t in (q, k, v)), {}), (tuple(t[0, 0] for t in (q, k, v)), {})]
    for args, kw in calls:
        want = _sdpa(*args, **kw)
        for same_length in (False, True):
            with pa.CrossAttnMode(same_length=same_length):
                assert torch.equal(_sdpa(*args, **kw), want)
    torch.manual_seed(11)
    want = _sdpa(q, k, v, dropout_p=0.25)
    torch.manual_seed(11)
    with pa.CrossAttnMode():
        assert torch.equal(_sdpa(q, k, v, dropout_p=0.25), want)
    # what it does compute is still its own, and what is wrong still raises
    mask = torch.rand(B, 1, 1, Skv, device="cuda", generator=g) < 0.7
    with pa.CrossAttnMode():
        assert torch.equal(_sdpa(q, k, v, attn_mask=mask, scale=0.25), ops.cross_attention(q, k, v, mask, scale=0.25))
        with pytest.raises(AssertionError, match="enable_gqa"):
            _sdpa(q, k[:, :1], v[:, :1])


def test_the_mode_does_not_lose_a_tangent():
    q, k, v = (t.float() for t in make(Sq=6, Skv=5))
    with fwAD.dual_level(), torch.nn.attention.sdpa_kernel(torch.nn.attention.SDPBackend.MATH):
        dual = fwAD.make_dual(q, torch.ones_like(q))
        want = fwAD.unpack_dual(_sdpa(dual, k, v)).tangent
        half = fwAD.make_dual(q.bfloat16(), torch.ones_like(q).bfloat16())
        want_half = fwAD.unpack_dual(_sdpa(half, k.bfloat16(), v.bfloat16())).tangent
        with pa.CrossAttnMode():
            assert torch.equal(fwAD.unpack_dual(_sdpa(dual, k, v)).tangent, want)
            assert torch.equal(fwAD.unpack_dual(_sdpa(half, k.bfloat16(), v.bfloat16())).tangent, want_half)
    assert math.isfinite(float(want.sum()))
