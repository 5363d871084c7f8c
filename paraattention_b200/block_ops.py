"""The differentiable operators around a transformer block's attention: cross attention to an
encoder's states (``cross_attention``) and the per-head norm of queries and keys with the position
rotation (``qk_norm_rotary``). Both are re-exported by :mod:`paraattention_b200.ops`.

Like the other ops of this package they are CUDA-only, launch on the current stream, never
synchronise, and raise instead of falling back. Both carry gradients: outside ``torch.no_grad()``,
with an input that requires a gradient, the call is recorded and its backward pass is a kernel of
libpa_b200 too (first derivatives only). Scratch memory comes from PyTorch's caching allocator per
call, so concurrent streams and captured graphs never share it.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import _status

__all__ = ["cross_attention", "qk_norm_rotary"]

_DTYPES = {torch.bfloat16: L.PA_BF16, torch.float16: L.PA_F16}


def _on(device: torch.device):
    """Makes ``device`` current for a launch (free when it already is)."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _ready(x: torch.Tensor) -> torch.Tensor:
    """x itself if the kernels can address it in place (unit stride on head_dim, 16-byte aligned base
    and strides, no broadcast dimensions), else a contiguous copy."""
    s0, s1, s2, s3 = x.stride()
    n0, n1, n2, _ = x.shape
    if (s3 == 1 and x.data_ptr() % 16 == 0 and (n0 == 1 or (s0 > 0 and s0 % 8 == 0))
            and (n1 == 1 or (s1 > 0 and s1 % 8 == 0)) and (n2 == 1 or (s2 > 0 and s2 % 8 == 0))):
        return x
    return x.clone(memory_format=torch.contiguous_format)  # (a contiguous view may still be misaligned)


def _strides(x: torch.Tensor):
    """(batch, head, row) element strides; those of dimensions of size 1 are never used: 0."""
    s = x.stride()
    n = x.shape
    return (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _bshd(shape, like: torch.Tensor) -> torch.Tensor:
    """[B, H, S, D] view of fresh [B, S, H, D] memory, the layout attention outputs have here."""
    b, h, s, d = shape
    return torch.empty((b, s, h, d), dtype=like.dtype, device=like.device).transpose(1, 2)


# ---- cross attention ---------------------------------------------------------------------------

def _check_cross(query, key, value, key_mask, scale):
    assert query.device.type == "cuda", "Must be CUDA tensors"
    assert query.ndim == 4 and key.ndim == 4 and value.ndim == 4, "query, key and value must be [B, H, S, D]"
    assert key.device == query.device and value.device == query.device, "query, key and value must be on one device"
    if query.dtype not in _DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
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


def _cross_args(q, k, v, rows, out, lse, scale) -> L.XattnArgs:
    a = L.XattnArgs()
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.batch, a.heads, a.seq_q, a.head_dim = q.shape
    a.kv_batch, a.kv_heads, a.seq_kv, _ = k.shape
    a.dtype = _DTYPES[q.dtype]
    a.scale = scale
    a.q_stride[:], a.k_stride[:], a.v_stride[:], a.o_stride[:] = _strides(q), _strides(k), _strides(v), _strides(out)
    if lse is not None:
        a.lse = lse.data_ptr()
    if rows is not None:
        a.key_mask = rows.data_ptr()
        a.mask_stride = rows.stride(0) if rows.shape[0] > 1 else 0
    return a


def _launch_cross(fn, a, backward, device):
    lib = L.load()
    with _on(device):
        n = lib.pa_xattn_workspace_bytes(C.byref(a), backward)
        if n < 0:
            L.check(int(n))
        if n > 0:
            ws = torch.empty(n, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        # The status word of this device: a wait that ran out in an earlier launch raises here. (It is made
        # on the first call; one that falls into a stream capture does without.)
        mirror = None
        if device.index in _status._single or not torch.cuda.is_current_stream_capturing():
            mirror = _status.single_gpu_status(device)
            mirror.check()
            a.status = mirror.word.data_ptr()
        L.check(fn(C.byref(a), torch.cuda.current_stream(device).cuda_stream))
        if mirror is not None and (backward or a.seq_q * (a.heads // a.kv_heads) > 16):
            mirror.refresh()  # (the kernel for few rows waits for nothing)


def _cross_forward(query, key, value, rows, scale, need_lse):
    B, Hq, Sq, D = query.shape
    out = _bshd(query.shape, query)
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=query.device) if need_lse else None
    if out.numel() == 0:
        return out, lse
    if key.shape[2] == 0:
        return out.zero_(), lse.fill_(-math.inf) if need_lse else None
    q, k, v = _ready(query), _ready(key), _ready(value)
    _launch_cross(L.load().pa_xattn_fwd, _cross_args(q, k, v, rows, out, lse, scale), 0, query.device)
    return out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, rows, scale):
        out, lse = _cross_forward(query, key, value, rows, scale, True)
        ctx.save_for_backward(query, key, value, rows, out, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        query, key, value, rows, out, lse = ctx.saved_tensors
        if dout is None:
            return None, None, None, None, None
        dq, dk, dv = _bshd(query.shape, query), _bshd(key.shape, key), _bshd(value.shape, value)
        if out.numel() == 0 or key.shape[2] == 0:
            return dq.zero_(), dk.zero_(), dv.zero_(), None, None
        q, k, v, g = _ready(query), _ready(key), _ready(value), _ready(dout)
        a = _cross_args(q, k, v, rows, out, lse, ctx.scale)
        a.dout, a.dq, a.dk, a.dv = g.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        a.do_stride[:], a.dq_stride[:], a.dk_stride[:], a.dv_stride[:] = _strides(g), _strides(dq), _strides(dk), _strides(dv)
        _launch_cross(L.load().pa_xattn_bwd, a, 1, query.device)
        return dq, dk, dv, None, None


def cross_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                    key_mask: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                    return_lse: bool = False):
    """Attention of ``query`` [B, Hq, Sq, D] to an encoder's states ``key``, ``value`` [B, Hkv, Skv, D]
    of another length: ``softmax(scale * query key^T) value``.

    ``Hq`` is a multiple of ``Hkv`` (shared key heads: query head h reads key head h // (Hq // Hkv));
    key and value may have batch size 1, one set of states for the whole batch. D is 64 or 128, bf16
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
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        out, lse = _CrossAttention.apply(query, key, value, rows, s)
        return (out, lse) if return_lse else out
    B = query.shape[0]
    if B > 1 and key.shape[0] == B and key.stride(0) == 0 and value.stride(0) == 0:
        key, value = key[:1], value[:1]  # (an expanded batch: read once)
    out, lse = _cross_forward(query, key, value, rows, s, return_lse)
    return (out, lse) if return_lse else out


# ---- norm and rotation of queries and keys --------------------------------------------------------

def _norm_args(xs, ys, weights, rotary, row_offset, interleaved, eps) -> L.QkNormArgs:
    a = L.QkNormArgs()
    x0 = xs[0]
    a.batch, _, a.rows, a.head_dim = x0.shape
    a.dtype = _DTYPES[x0.dtype]
    a.interleaved = 1 if interleaved else 0
    a.eps = eps
    for i, (x, y, w) in enumerate(zip(xs, ys, weights)):
        a.x[i], a.y[i] = x.data_ptr(), y.data_ptr()
        a.heads[i] = x.shape[1]
        (a.x_stride[i][0], a.x_stride[i][2], a.x_stride[i][1]) = _strides(x)
        (a.y_stride[i][0], a.y_stride[i][2], a.y_stride[i][1]) = _strides(y)
        if w is not None:
            a.weight[i] = w.data_ptr()
    if rotary is not None:
        a.cos, a.sin = rotary[0].data_ptr(), rotary[1].data_ptr()
        a.table_row0 = row_offset
    return a


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=torch.contiguous_format)


def _norm_forward(xs, weights, rotary, row_offset, interleaved, eps):
    ys = [_bshd(x.shape, x) for x in xs]
    if ys[0].numel() == 0:
        return ys
    a = _norm_args([_ready(x) for x in xs], ys, [_aligned(w) for w in weights], rotary, row_offset, interleaved, eps)
    with _on(xs[0].device):
        L.check(L.load().pa_qk_norm_fwd(C.byref(a), torch.cuda.current_stream(xs[0].device).cuda_stream))
    return ys


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, row_offset, interleaved, eps):
        xs = [q] if k is None else [q, k]
        rotary = None if cos is None else (cos, sin)
        ys = _norm_forward(xs, (q_weight, k_weight), rotary, row_offset, interleaved, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin)
        ctx.plan = (row_offset, interleaved, eps)
        return (ys[0], None) if k is None else tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin = ctx.saved_tensors
        row_offset, interleaved, eps = ctx.plan
        grads = [None] * 9
        need = ctx.needs_input_grad
        # the tensors something is asked of: (x, weight, dy, index of x among the inputs, of the weight)
        parts = [(x, w, g, i, i + 2) for i, (x, w, g) in enumerate(((q, q_weight, dq_out), (k, k_weight, dk_out)))
                 if x is not None and (need[i] or need[i + 2])]
        if not parts:
            return tuple(grads)
        xs, dys = [_ready(p[0]) for p in parts], [_ready(p[2]) for p in parts]
        dxs = [_bshd(x.shape, x) for x in xs]
        ws = [_aligned(p[1]) for p in parts]
        dws = [torch.empty_like(w) if w is not None and need[p[4]] else None for w, p in zip(ws, parts)]
        if xs[0].numel() == 0:
            dws = [w if w is None else w.zero_() for w in dws]
        else:
            a = _norm_args(xs, dxs, ws, None if cos is None else (cos, sin), row_offset, interleaved, eps)
            device = xs[0].device
            lib = L.load()
            with _on(device):
                for i, (g, dw) in enumerate(zip(dys, dws)):
                    a.dy[i] = g.data_ptr()
                    (a.dy_stride[i][0], a.dy_stride[i][2], a.dy_stride[i][1]) = _strides(g)
                    if dw is not None:
                        a.dweight[i] = dw.data_ptr()
                if any(w is not None for w in dws):
                    scratch = torch.empty(lib.pa_qk_norm_workspace_bytes(), dtype=torch.uint8, device=device)
                    a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
                L.check(lib.pa_qk_norm_bwd(C.byref(a), torch.cuda.current_stream(device).cuda_stream))
        for p, dx, dw in zip(parts, dxs, dws):
            if need[p[3]]:
                grads[p[3]] = dx
            grads[p[4]] = dw
        return tuple(grads)


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
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
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
        cos, sin = _aligned(cos), _aligned(sin)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, row_offset, interleaved, eps)
    ys = _norm_forward([q] if k is None else [q, k], (q_weight, k_weight), None if cos is None else (cos, sin), row_offset,
                       interleaved, eps)
    return (ys[0], None) if k is None else tuple(ys)
