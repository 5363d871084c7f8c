"""No-GPU check of what pa.CrossAttnMode hands on: calls in a form that cross_attn_func does not compute."""
import pytest
import torch
import torch.nn.functional as F

import paraattention_b200 as pa


def test_calls_in_other_forms_are_handed_on():
    q, k = torch.randn(2, 2, 8, 64), torch.randn(2, 2, 5, 64)
    calls = [((q, k, k), {"attn_mask": torch.randn(2, 1, 1, 5)}), ((q, k, k), {"attn_mask": torch.rand(2, 1, 8, 5) < 2.0}),
             ((q, k, k), {"is_causal": True}), ((q[0], k[0], k[0]), {}), ((q[0, 0], k[0, 0], k[0, 0]), {})]
    for args, kw in calls:
        want = F.scaled_dot_product_attention(*args, **kw)
        for same_length in (False, True):
            with pa.CrossAttnMode(same_length=same_length):
                assert torch.equal(F.scaled_dot_product_attention(*args, **kw), want)
                named = dict(zip(("query", "key", "value"), args), **kw)
                assert torch.equal(F.scaled_dot_product_attention(**named), want)
    torch.manual_seed(3)
    want = F.scaled_dot_product_attention(q, k, k, dropout_p=0.5)
    torch.manual_seed(3)
    with pa.CrossAttnMode():
        assert torch.equal(F.scaled_dot_product_attention(q, k, k, dropout_p=0.5), want)


def test_handed_on_calls_reach_the_mode_around():
    seen = []

    class Outer(pa.CrossAttnMode):
        def _call_attn_func(self, *args, **kwargs):
            seen.append(kwargs)
            return args[0]

    q, k = torch.randn(2, 2, 8, 64), torch.randn(2, 2, 5, 64)
    with Outer(), pa.CrossAttnMode():
        out = F.scaled_dot_product_attention(q, k, k, dropout_p=0.5)
    assert out is q and seen == [{"dropout_p": 0.5}]


def test_wrong_arguments_still_raise():
    q, k = torch.randn(2, 2, 8, 64), torch.randn(2, 2, 5, 64)
    with pa.CrossAttnMode():
        with pytest.raises(AssertionError, match="enable_gqa"):
            F.scaled_dot_product_attention(q, k[:, :1], k[:, :1])
        with pytest.raises(AssertionError, match="CUDA"):
            F.scaled_dot_product_attention(q, k, k)
