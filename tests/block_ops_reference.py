"""64-bit references of cross attention and of the q/k norm with rotation, and elementwise bounds on
how far a correct 16-bit result may be from them.

Bounds. u = half a unit in the last place of the tensors' type relative to the value (bf16 2^-8 / 2 ...
torch.finfo(t).eps / 2). The kernels round P (and dS) to the type once and the results once; all else
is fp32, for which SLACK = 2^-13 of the absolute sums is allowed (products of 128 terms and sums over
a few thousand keys stay below 2^-14, the approximate exponential adds 2^-22).

  out: P relative error u -> u * A with A = W |V|; final rounding u |out| <= u A.       (2 u + SLACK) A
  delta: sum do * out, out as above -> E = sum_d |do| (2 u + SLACK) A
  dS = P (dP - delta): u |dS| + P E + SLACK P (|do| |V|^T)
  dv: (2 u + SLACK) P^T |do|;  dk, dq: the dS error times |q| or |k|, plus the final rounding u |result|
"""
import math

import torch

SLACK = 2.0 ** -13


def unit(t):
    return torch.finfo(t).eps / 2


def cross_reference(q, k, v, mask=None, scale=None, do=None):
    """(values, bounds) in float64: out, lse and with do also dq, dk, dv. k, v may have batch 1 and fewer heads."""
    u = unit(q.dtype)
    B, Hq, Sq, D = q.shape
    Bk, Hk, Skv, _ = k.shape
    G = Hq // Hk
    s = 1.0 / math.sqrt(D) if scale is None else scale
    q64 = q.detach().double()
    ke, ve = (t.detach().double().expand(B, -1, -1, -1).repeat_interleave(G, dim=1) for t in (k, v))
    keep = torch.ones(B, 1, 1, Skv, dtype=torch.bool, device=q.device) if mask is None else mask.expand(B, Skv)[:, None, None, :]
    clean = keep.transpose(-1, -2)  # [B, 1, Skv, 1]
    ke, ve = torch.where(clean, ke, 0.0), torch.where(clean, ve, 0.0)
    z = torch.einsum("bhmd,bhnd->bhmn", q64, ke) * s
    za = torch.einsum("bhmd,bhnd->bhmn", q64.abs(), ke.abs()) * s
    z = z.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(z, dim=-1) if Skv else torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.where(lse[..., None] == -math.inf, 0.0, torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)[..., None]))
    out = w @ ve
    A = w @ ve.abs()
    vals = {"out": out, "lse": lse}
    bound = {"out": (2 * u + SLACK) * A,
             "lse": 2.0 ** -18 * za.amax(dim=-1) + 1e-5 if Skv else torch.zeros_like(lse)}
    if do is None:
        return vals, bound
    g = do.double()
    dp = torch.einsum("bhmd,bhnd->bhmn", g, ve)
    dpa = torch.einsum("bhmd,bhnd->bhmn", g.abs(), ve.abs())
    ds = w * (dp - (g * out).sum(-1, keepdim=True))
    E = (g.abs() * bound["out"]).sum(-1, keepdim=True)
    eds = u * ds.abs() + w * E + SLACK * w * (dpa + (g.abs() * A).sum(-1, keepdim=True))

    def to_keys(x):  # [B, Hq, Skv, D] -> [Bk, Hk, Skv, D]
        x = x.reshape(B, Hk, G, Skv, D).sum(2)
        return x.sum(0, keepdim=True) if Bk == 1 else x

    vals["dq"] = s * torch.einsum("bhmn,bhnd->bhmd", ds, ke)
    vals["dk"] = to_keys(s * torch.einsum("bhmn,bhmd->bhnd", ds, q64))
    vals["dv"] = to_keys(torch.einsum("bhmn,bhmd->bhnd", w, g))
    bound["dq"] = s * torch.einsum("bhmn,bhnd->bhmd", eds, ke.abs()) + u * vals["dq"].abs()
    bound["dk"] = to_keys(s * torch.einsum("bhmn,bhmd->bhnd", eds, q64.abs())) + u * vals["dk"].abs()
    bound["dv"] = to_keys((2 * u + SLACK) * torch.einsum("bhmn,bhmd->bhnd", w, g.abs()))
    return vals, bound


def norm_reference(x, w, rotary, interleaved, eps, row_offset=0, dy=None):
    """(values, bounds) of y and with dy also dx, dw. One rounding each: u |value|, plus fp32 slack of 2^-18 of
    the absolute sums (an fp32 sum of 128 squares, a reciprocal square root, two products)."""
    u, tiny = unit(x.dtype), 2.0 ** -18
    D = x.shape[-1]
    x64 = x.detach().double()
    w64 = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    r = 1.0 if w is None else 1.0 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    n = x64 * r

    def turn(t, back=False, absolute=False):
        if rotary is None:
            return t.abs() if absolute else t
        cos, sin = (m[row_offset:row_offset + x.shape[2]].double() for m in rotary)
        if absolute:
            cos, sin, t = cos.abs(), sin.abs(), t.abs()
        first = slice(0, D, 2) if interleaved else slice(0, D // 2)
        second = slice(1, D, 2) if interleaved else slice(D // 2, D)
        a, c = t[..., first], t[..., second]
        o = torch.empty_like(t)
        sg = 1.0 if absolute else -1.0
        if back:
            o[..., first] = a * cos[:, first] + c * sin[:, second]
            o[..., second] = c * cos[:, second] + sg * a * sin[:, first]
        else:
            o[..., first] = a * cos[:, first] + sg * c * sin[:, first]
            o[..., second] = c * cos[:, second] + a * sin[:, second]
        return o

    y = turn(n * w64)
    vals = {"y": y}
    # (the smallest 16-bit numbers are spaced absolutely, not relatively: f16 subnormals are 2^-24 apart)
    floor = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    bound = {"y": u * y.abs() + tiny * turn(n * w64, absolute=True) + floor}
    if dy is None:
        return vals, bound
    uu = turn(dy.double(), back=True)
    ua = turn(dy.double(), back=True, absolute=True)
    g, ga = uu * w64, ua * w64.abs()
    if w is None:
        vals["dx"], bound["dx"] = uu, u * uu.abs() + tiny * ua + floor
        return vals, bound
    vals["dx"] = r * (g - n * (g * n).mean(-1, keepdim=True))
    bound["dx"] = u * vals["dx"].abs() + tiny * r * (ga + n.abs() * (ga * n.abs()).mean(-1, keepdim=True)) + floor
    vals["dw"] = (uu * n).sum(dim=(0, 1, 2))
    bound["dw"] = u * vals["dw"].abs() + tiny * (ua * n.abs()).sum(dim=(0, 1, 2)) + floor
    return vals, bound


def assert_within(got, want, bound, what):
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    same = got == want  # (infinities)
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= bound) & ~same
    if bool(bad.any()):
        i = int(torch.where(bad.flatten(), (off - bound).flatten().nan_to_num(math.inf), -1.0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bounds; worst at {i}: "
                             f"{float(got.flatten()[i])} against {float(want.flatten()[i])} +- {float(bound.flatten()[i])}")
