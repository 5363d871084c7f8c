"""The differentiable operators around a transformer block's attention: cross attention to an
encoder's states (``cross_attention``) and the per-head norm of queries and keys with the position
rotation (``qk_norm_rotary``). Both are re-exported by :mod:`paraattention_b200.ops`.

Like the other ops of this package they are CUDA-only, launch on the current stream, never
synchronise, and raise instead of falling back. Both carry gradients: outside ``torch.no_grad()``,
with an input that requires a gradient, the call is recorded and its backward pass is a kernel of
libpa_b200 too (first derivatives in reverse mode only; a tensor with a forward-mode tangent is
refused). The arguments are checked here; the rest of a call - output and scratch memory from
PyTorch's caching allocator (so concurrent streams and captured graphs never share scratch), the C
ABI's argument structures, the autograd node - is the extension _pa_torch.so (csrc/pa_torch.cpp).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib as L
from . import _status

__all__ = ["cross_attention", "qk_norm_rotary"]

_TYPES = (torch.bfloat16, torch.float16)


def _status_addresses(device: torch.device) -> Tuple[int, int]:
    """Addresses of this device's status word and of its pinned mirror (made on the first call; one that
    falls into a stream capture does without: (0, 0))."""
    m = _status._single.get(device.index)
    if m is None:
        if torch.cuda.is_current_stream_capturing():
            return 0, 0
        m = _status.single_gpu_status(device)
    return m.word.data_ptr(), m.host.data_ptr()


# ---- cross attention ---------------------------------------------------------------------------

def _check_cross(query, key, value, key_mask, scale):
    assert query.device.type == "cuda", "Must be CUDA tensors"
    assert query.ndim == 4 and key.ndim == 4 and value.ndim == 4, "query, key and value must be [B, H, S, D]"
    assert key.device == query.device and value.device == query.device, "query, key and value must be on one device"
    if query.dtype not in _TYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        raise NotImplementedError(f"cross_attention dtype {query.dtype}: only bfloat16 and float16 are built "
                                  "(query, key and value alike)")
    B, Hq, _, D = query.shape
    if D not in (64, 128) or key.shape[-1] != D or value.shape[-1] != D:
        raise NotImplementedError(f"head_dim {D}: only 64 and 128 are built (query, key and value alike)")
    assert value.shape == key.shape, "key and value must have the same shape"
    assert key.shape[0] in (1, B), f"batch of key and value must be {B} or 1, not {key.shape[0]}"
    assert key.shape[1] > 0 and Hq % key.shape[1] == 0, \
        f"{Hq} query heads are not a multiple of {key.shape[1]} key heads"
    if scale is not None and not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if key_mask is None:
        return None
    from .ops import key_mask_of

    assert key_mask.dtype == torch.bool, "key_mask must be a boolean tensor"
    assert key_mask.device == query.device, "key_mask must be on the same device"
    # [B, Skv] or [1, Skv] per batch entry; the 4-D form of attention masks; one row for all
    rows = key_mask[:, None, None, :] if key_mask.ndim == 2 else key_mask
    rows = key_mask_of(rows, B, key.shape[2])
    if rows is None:
        raise NotImplementedError(f"key_mask of shape {tuple(key_mask.shape)}: expected a key-padding mask "
                                  f"[{B}, {key.shape[2]}] or broadcastable to [{B}, 1, 1, {key.shape[2]}]")
    if rows.stride(1) != 1 and rows.shape[1] > 1:
        rows = rows.contiguous()
    return rows


def cross_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                    key_mask: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    return_lse: bool = False):
    """Attention of ``query`` [B, Hq, Sq, D] to an encoder's states ``key``, ``value`` [B, Hkv, Skv, D]
    of another length: ``softmax(scale * query key^T) value``.

    ``Hq`` is a multiple of ``Hkv`` (shared key heads: query head h reads key head h // (Hq // Hkv));
    key and value may have batch size 1, one set of states for the whole batch: with gradients, that is the form to
    give them in. (States expanded to the batch are copied once per batch entry then, in the forward and in the
    backward pass, and PyTorch adds up the entries' gradients in 16 bits.) D is 64 or 128, bf16
    or f16, any strides. ``key_mask``: boolean, True = the key takes part, [B, Skv] or [1, Skv] (or an
    attention mask broadcastable to [B, 1, 1, Skv]); what masked keys and values hold does not matter.
    A query without any key gets zeros (and an LSE of -inf, and no gradient). ``scale`` defaults to
    1 / sqrt(D) and must be positive.

    Returns the output, a [B, Hq, Sq, D] view of [B, Sq, Hq, D] memory, or with ``return_lse`` also
    the natural log-sum-exp of the logits, fp32 [B, Hq, Sq] (which carries no gradient). Gradients of
    query, key and value are computed by libpa_b200; they are sums in a fixed order, so equal calls
    give equal results. A backward pass that is captured into a CUDA graph has to own its autograd
    graph, as PyTorch asks: no eager graph over the same leaves may be alive during the capture."""
    rows = _check_cross(query, key, value, key_mask, scale)
    s = 1.0 / math.sqrt(query.shape[-1]) if scale is None else float(scale)
    out, lse = L.load_torch_ext().cross_attention(query, key, value, rows, s, return_lse, *_status_addresses(query.device))
    return (out, lse) if return_lse else out


# ---- norm and rotation of queries and keys --------------------------------------------------------

def qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None,
                   rotary: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, *, eps: float = 1e-6,
                   interleaved: bool = True, row_offset: int = 0):
    """Per-head RMSNorm of ``q`` [B, Hq, S, D] and ``k`` [B, Hk, S, D] and the rotation of their positions,
    in one launch: ``R(row) (weight * x / sqrt(mean(x^2) + eps))``, computed in fp32 and rounded once.

    The differentiable relative of ``qkv_prepare`` (which rounds where the eager sequence rounds and
    places v too): gradients of q, k and both weights. Head counts of q and k may differ; k may be
    None. Weights: [D] in the tensors' dtype, or None: no norm. ``rotary = (cos, sin)``: fp32
    [rows, D] tables of which row ``row_offset + s`` belongs to row s, or None: no rotation; the tables
    carry no gradient. Pairs are the adjacent elements (2i, 2i + 1), or with ``interleaved=False``
    (i, i + D / 2); a pair (a, c) becomes (a cos_a - c sin_a, c cos_c + a sin_c). D is 64 or 128, bf16 or
    f16, any strides. Returns (q_out, k_out), [B, H, S, D] views of [B, S, H, D] memory (k_out is None
    without k)."""
    assert q.device.type == "cuda", "Must be CUDA tensors"
    assert q.ndim == 4 and (k is None or k.ndim == 4), "q and k must be [B, H, S, D]"
    if q.dtype not in _TYPES or (k is not None and k.dtype != q.dtype):
        raise NotImplementedError(f"qk_norm_rotary dtype {q.dtype}: only bfloat16 and float16 are built (q and k alike)")
    B, _, S, D = q.shape
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: only 64 and 128 are built")
    assert k is None or (k.shape[0] == B and k.shape[2] == S and k.shape[3] == D), \
        "q and k must agree in batch, rows and head_dim"
    assert k is None or k.device == q.device, "q and k must be on one device"
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, not {eps}")
    for w in (q_weight, k_weight):
        assert w is None or (w.shape == (D,) and w.dtype == q.dtype and w.device == q.device), \
            f"weights must be [{D}] in the dtype and on the device of q"
    assert k is not None or k_weight is None, "k_weight without k"
    cos = sin = None
    if rotary is not None:
        cos, sin = rotary
        assert cos.dtype == torch.float32 and sin.dtype == torch.float32, "cos and sin must be fp32"
        assert cos.shape == sin.shape and cos.ndim == 2 and cos.shape[1] == D, f"cos and sin must be [rows, {D}] alike"
        assert row_offset >= 0 and cos.shape[0] >= row_offset + S, "the tables end before the last row"
        assert cos.device == q.device and sin.device == q.device, "cos and sin must be on the device of q"
        if cos.requires_grad or sin.requires_grad:
            raise NotImplementedError("qk_norm_rotary computes no gradient of cos and sin")
    return L.load_torch_ext().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, row_offset, interleaved, eps)
