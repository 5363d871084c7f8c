"""Cases of the attention neighbours of a transformer block: cross attention to an encoder's states
(forward, padded prompts, shared key/value heads, single tokens, training) and the per-head norm of
queries and keys with the position rotation (forward, training).

``run`` computes the plain form in 32 bits with elementary tensor operations, or - with ``own`` - calls
the framework: ``ops.cross_attention`` and ``ops.qk_norm_rotary``. ``exact`` states the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _cross(name, b, hq, hkv, sq, skv, d, dtype, train=False, lens="", lse=False):
    return {"name": name, "op": "cross", "b": b, "hq": hq, "hkv": hkv, "sq": sq, "skv": skv, "d": d, "dtype": dtype,
            "train": train, "lens": lens, "lse": lse}


def _norm(name, b, hq, hkv, s, d, dtype, train=False, interleaved=True):
    return {"name": name, "op": "norm", "b": b, "hq": hq, "hkv": hkv, "sq": s, "d": d, "dtype": dtype, "train": train,
            "interleaved": interleaved}


def listed():
    return [
        # every video token of a 480x832, 81-frame clip attends to a 512-token prompt (one block, one denoising step)
        _cross("video_to_prompt", 1, 40, 40, 32760, 512, 128, "bf16"),
        # the same block in a fine-tuning step: output and the gradients of queries, keys and values
        _cross("video_to_prompt_train", 1, 40, 40, 32760, 512, 128, "bf16", train=True),
        # image tokens, a batch of prompts padded to 512, one of them empty (dropped for guidance)
        _cross("image_padded_prompts", 4, 24, 24, 4096, 512, 128, "bf16", lens="0.14,0,0.6,1", lse=True),
        # short text encoder of 77 tokens, odd rows, head_dim 64, fine-tuning
        _cross("short_prompt_train", 2, 16, 16, 1000, 77, 64, "f16", train=True),
        # shared key/value heads, padded prompts, fine-tuning
        _cross("shared_heads_padded_train", 2, 32, 8, 2049, 333, 128, "bf16", train=True, lens="0.35,1"),
        # one token per sequence against its encoder's states (autoregressive decoder), padded
        _cross("single_tokens", 64, 32, 8, 1, 2048, 128, "bf16", lens="1,0.75,0.5,0.9"),
        # the smallest call: one token, one short prompt - latency
        _cross("single_token_short_prompt", 1, 24, 24, 1, 77, 128, "f16", lse=True),
        # a few learned queries gather a whole clip: few rows, long keys
        _cross("queries_to_video", 1, 24, 24, 256, 32760, 128, "bf16", lse=True),
        # q and k of one joint-attention call: 512 text + 4096 image tokens
        _norm("joint_qk", 1, 24, 24, 4608, 128, "bf16"),
        # q and k of a clip in a fine-tuning step: outputs, gradients of q, k and both weights
        _norm("video_qk_train", 1, 40, 40, 32760, 128, "bf16", train=True),
        # one new token per sequence, shared key heads, half-split pairs - latency
        _norm("single_token_qk", 8, 32, 8, 1, 64, "f16", interleaved=False),
        # odd rows, shared key heads, half-split pairs, fine-tuning
        _norm("odd_qk_train", 2, 32, 8, 1001, 64, "f16", train=True, interleaved=False),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; odd ones as likely as even ones."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    d = rng.choice((64, 128))
    dtype = rng.choice(("bf16", "f16"))
    hkv = rng.choice((1, 2, 3, 5, 8, 12, 24, 40))
    group = rng.choice((1, 1, 1, 2, 4, 8)) if hkv <= 8 else 1
    b = rng.choice((1, 1, 2, 3, 4, 8, 16))
    train = rng.random() < 0.5
    if rng.random() < 0.3:
        most = 32760 * 40 // max(1, b * hkv * group)
        return {k: v for k, v in _norm("", b, hkv * group, hkv, _spread(rng, 1, max(1, min(32760, most))), d, dtype, train,
                                       rng.random() < 0.5).items() if k != "name"}
    sq = _spread(rng, 16 if train else 1, 32760)
    skv = _spread(rng, 16 if train else 1, 2048 if sq > 256 else 32760)
    while b * hkv * group * sq * skv > 40 * 32760 * 512 or b * hkv * group * max(sq, skv) > 40 * 32760:
        if b > 1:
            b -= 1
        elif hkv > 1:
            hkv -= 1
        elif group > 1:
            group //= 2
        else:
            sq = max(16, sq // 2)
    lens = ""
    if rng.random() < 0.5:
        lens = ",".join("%.2f" % rng.choice((1.0, 1.0, 0.0 if i else 0.9, rng.uniform(0.2 if i else 0.6, 1.0))) for i in range(b))
    return {k: v for k, v in _cross("", b, hkv * group, hkv, sq, skv, d, dtype, train, lens, not train and rng.random() < 0.5).items()
            if k != "name"}


def _lengths(case):
    if not case["lens"]:
        return [case["skv"]] * case["b"]
    fractions = [float(x) for x in case["lens"].split(",")]
    return [int(round(fractions[i % len(fractions)] * case["skv"])) for i in range(case["b"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(t)

    b, hq, hkv, sq, d = case["b"], case["hq"], case["hkv"], case["sq"], case["d"]
    s = {"case": case}
    if case["op"] == "cross":
        skv = case["skv"]
        # projection outputs viewed per head: [B, H, S, D] views of [B, S, H, D] memory
        s["q"] = normal(b, sq, hq, d).transpose(1, 2)
        s["k"] = normal(b, skv, hkv, d).transpose(1, 2)
        s["v"] = normal(b, skv, hkv, d).transpose(1, 2)
        s["mask"] = None
        if case["lens"]:
            lens = torch.tensor(_lengths(case), device="cuda")[torch.randperm(b, generator=g, device="cuda")]
            s["mask"] = torch.arange(skv, device="cuda")[None, :] < lens[:, None]
        if case["train"]:
            s["do"] = normal(b, sq, hq, d).transpose(1, 2)
        names = ("q", "k", "v")
    else:
        s["q"] = normal(b, sq, hq, d, scale=2.0).transpose(1, 2)
        s["k"] = normal(b, sq, hkv, d, scale=2.0).transpose(1, 2)
        s["wq"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(t)
        s["wk"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(t)
        freq = torch.exp(torch.arange(0, d, 2, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / d))
        first = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
        ang = (first + torch.arange(sq, device="cuda", dtype=torch.float64))[:, None] * freq
        ang = ang.repeat_interleave(2, dim=-1) if case["interleaved"] else torch.cat([ang, ang], dim=-1)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        if case["train"]:
            s["dq"] = normal(b, sq, hq, d).transpose(1, 2)
            s["dk"] = normal(b, sq, hkv, d).transpose(1, 2)
        names = ("q", "k", "wq", "wk")
    if case["train"]:
        for n in names:
            s[n].requires_grad_(True)
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _grouped(x, hkv):
    """[B, Hq, S, D] -> [B, Hkv, group * S, D] in 32 bits: the rows that share a key/value head."""
    b, hq, s, d = x.shape
    return x.detach().float().reshape(b, hkv, hq // hkv * s, d)


def _plain_cross(s):
    c = s["case"]
    b, hq, hkv, sq, d = c["b"], c["hq"], c["hkv"], c["sq"], c["d"]
    t = s["q"].dtype
    scale = 1.0 / math.sqrt(d)
    q, k, v = _grouped(s["q"], hkv), s["k"].detach().float(), s["v"].detach().float()
    logits = (q @ k.transpose(-1, -2)) * scale
    if s["mask"] is not None:
        logits = logits.masked_fill(~s["mask"][:, None, None, :], -math.inf)
    top = logits.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(logits - top)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    out = o.reshape(b, hq, sq, d).to(t)
    if not c["train"]:
        return (out, (torch.log(total) + top).reshape(b, hq, sq)) if c["lse"] else out
    do = _grouped(s["do"], hkv)
    dv = p.transpose(-1, -2) @ do
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(dim=-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q) * scale
    return out, dq.reshape(b, hq, sq, d).to(t), dk.to(t), dv.to(t)


def _turn(x, cos, sin, interleaved, back=False):
    """The rotation of pairs (adjacent elements, or element i with i + D/2), or its transpose."""
    d = x.shape[-1]
    if interleaved:
        a, c = x[..., 0::2], x[..., 1::2]
        ca, sa, cc, sc = cos[:, 0::2], sin[:, 0::2], cos[:, 1::2], sin[:, 1::2]
    else:
        a, c = x[..., : d // 2], x[..., d // 2:]
        ca, sa, cc, sc = cos[:, : d // 2], sin[:, : d // 2], cos[:, d // 2:], sin[:, d // 2:]
    if back:
        ya, yc = a * ca + c * sc, c * cc - a * sa
    else:
        ya, yc = a * ca - c * sa, c * cc + a * sc
    return torch.stack([ya, yc], dim=-1).flatten(-2) if interleaved else torch.cat([ya, yc], dim=-1)


def _plain_norm_one(s, x, w, dy):
    c = s["case"]
    t = x.dtype
    x, w = x.detach().float(), w.detach().float()
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6)
    n = x * r
    y = _turn(n * w, s["cos"], s["sin"], c["interleaved"]).to(t)
    if dy is None:
        return y
    u = _turn(dy.float(), s["cos"], s["sin"], c["interleaved"], back=True)
    g = u * w
    dx = r * (g - n * (g * n).mean(dim=-1, keepdim=True))
    return y, dx.to(t), (u * n).sum(dim=(0, 1, 2)).to(t)


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    if own:
        from paraattention_b200 import ops
        if c["op"] == "cross":
            if c["train"]:
                out = ops.cross_attention(state["q"], state["k"], state["v"], state["mask"])
                return (out.detach(),) + torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"])
            return ops.cross_attention(state["q"], state["k"], state["v"], state["mask"], return_lse=c["lse"])
        yq, yk = ops.qk_norm_rotary(state["q"], state["k"], state["wq"], state["wk"], (state["cos"], state["sin"]),
                                    eps=1e-6, interleaved=c["interleaved"])
        if not c["train"]:
            return yq, yk
        dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), (state["q"], state["k"], state["wq"], state["wk"]),
                                               (state["dq"], state["dk"]))
        return yq.detach(), dq, dwq, yk.detach(), dk, dwk
    if c["op"] == "cross":
        return _plain_cross(state)
    if not c["train"]:
        return _plain_norm_one(state, state["q"], state["wq"], None), _plain_norm_one(state, state["k"], state["wk"], None)
    return (_plain_norm_one(state, state["q"], state["wq"], state["dq"])
            + _plain_norm_one(state, state["k"], state["wk"], state["dk"]))


def work(case):
    b, hq, hkv, sq, d = case["b"], case["hq"], case["hkv"], case["sq"], case["d"]
    if case["op"] == "cross":
        keys = sum(_lengths(case))
        rows, kv = 2.0 * b * hq * sq * d, 2.0 * keys * hkv * d
        flops = 4.0 * hq * sq * keys * d
        if case["train"]:  # q, do in; out, dq out; k, v in; dk, dv out (whole, padding included)
            return {"bytes": 4 * rows + 2 * kv + 4.0 * b * case["skv"] * hkv * d, "flops": 3.5 * flops}
        return {"bytes": 2 * rows + 2 * kv + (4.0 * b * hq * sq if case["lse"] else 0), "flops": flops}
    n = float(b) * (hq + hkv) * sq * d
    tables = 8.0 * sq * d
    return {"bytes": (8 if case["train"] else 4) * n + tables, "flops": (22 if case["train"] else 8) * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_cross(case, s):
    b, hq, hkv, sq, d = case["b"], case["hq"], case["hkv"], case["sq"], case["d"]
    skv, group = case["skv"], hq // hkv
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, dq, lse = new(b, hq, sq, d), new(b, hq, sq, d) if case["train"] else None, torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device="cuda")
    dk, dv = (new(b, hkv, skv, d), new(b, hkv, skv, d)) if case["train"] else (None, None)
    for i in range(b):
        keep = torch.arange(skv, device="cuda") if s["mask"] is None else s["mask"][i].nonzero()[:, 0]
        if keep.numel() == 0:
            continue
        for h in range(hq):
            q = s["q"][i, h].detach().double() / math.sqrt(d)
            k, v = s["k"][i, h // group].detach().double()[keep], s["v"][i, h // group].detach().double()[keep]
            z = torch.einsum("md,nd->mn", q, k)
            lse[i, h] = torch.logsumexp(z, dim=1)
            w = torch.softmax(z, dim=1)
            out[i, h] = torch.einsum("mn,nd->md", w, v)
            if case["train"]:
                g = s["do"][i, h].double()
                dw = torch.einsum("md,nd->mn", g, v)
                dz = w * (dw - torch.einsum("mn,mn->m", dw, w)[:, None])
                dq[i, h] = torch.einsum("mn,nd->md", dz, k) / math.sqrt(d)
                dk[i, h // group].index_add_(0, keep, torch.einsum("mn,md->nd", dz, q))
                dv[i, h // group].index_add_(0, keep, torch.einsum("mn,md->nd", w, g))
    if case["train"]:
        return out, dq, dk, dv
    return (out, lse) if case["lse"] else out


def _exact_norm(case, s, x, w, dy):
    d = case["d"]
    x, w = x.detach().double(), w.detach().double()
    cos, sin = s["cos"].double(), s["sin"].double()
    even = torch.arange(0, d, 2, device="cuda") if case["interleaved"] else torch.arange(d // 2, device="cuda")
    odd = even + (1 if case["interleaved"] else d // 2)
    # the rotation of every row as a matrix [S, D, D]
    m = torch.zeros(case["sq"], d, d, dtype=torch.float64, device="cuda")
    m[:, even, even], m[:, even, odd] = cos[:, even], -sin[:, even]
    m[:, odd, odd], m[:, odd, even] = cos[:, odd], sin[:, odd]
    size = torch.sqrt(x.square().sum(dim=-1, keepdim=True) / d + 1e-6)
    y = torch.einsum("bhsj,sij->bhsi", x / size * w, m)
    if dy is None:
        return y
    u = torch.einsum("bhsi,sij->bhsj", dy.double(), m)
    dx = u * w / size - x * (u * w * x).sum(dim=-1, keepdim=True) / (d * size ** 3)
    return y, dx, torch.einsum("bhsj,bhsj->j", u, x / size)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "cross":
            return _exact_cross(case, s)
        if not case["train"]:
            return _exact_norm(case, s, s["q"], s["wq"], None), _exact_norm(case, s, s["k"], s["wk"], None)
        return _exact_norm(case, s, s["q"], s["wq"], s["dq"]) + _exact_norm(case, s, s["k"], s["wk"], s["dk"])
