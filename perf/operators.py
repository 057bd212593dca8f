"""The operators of the text encoder's blocks, as cases to be measured: root-mean-square norm of a residual stream, self-attention with a
learned relative position bias, and the gated feed-forward product.

`run` computes them in their plain form (elementary torch operations in 32 bits) or, where `own` is set, through aether_amd.ops.
"""
import math

import torch

own = False

#: values of one e4m3 number are at most this
E4M3_MAX = 448.0


# ---- cases ---------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one prompt of the transformer's text length through a block's norm: the residual stream is fp32, the block's output (delta) bf16
        dict(name="norm_prompt", op="rms_norm", mode="infer", rows=226, dim=4096, stream="float32"),
        # 64 prompts, output in 8 bits for the feed-forward's 8-bit weights
        dict(name="norm_batch_e4m3", op="rms_norm", mode="e4m3", rows=14464, dim=4096, stream="float32"),
        # a training step on 16 prompts: forward, then the gradients of stream, delta and weight
        dict(name="norm_train", op="rms_norm", mode="train", rows=3616, dim=4096, stream="float32"),
        # a short prompt without padding: the smallest call, where latency counts
        dict(name="attn_short", op="relbias_attn", mode="infer", batch=1, length=19, heads=64, buckets=32, max_distance=128, ragged=False),
        # 16 prompts of different lengths, padded to the text length
        dict(name="attn_prompts", op="relbias_attn", mode="infer", batch=16, length=226, heads=64, buckets=32, max_distance=128, ragged=True),
        # a long document, odd length
        dict(name="attn_long", op="relbias_attn", mode="infer", batch=1, length=7993, heads=16, buckets=32, max_distance=128, ragged=False),
        # a training step on 16 padded prompts: forward, then the gradients of q, k, v and the bias table
        dict(name="attn_train_prompts", op="relbias_attn", mode="train", batch=16, length=226, heads=64, buckets=32, max_distance=128, ragged=True),
        # a training step on two long texts of odd length
        dict(name="attn_train_long", op="relbias_attn", mode="train", batch=2, length=2039, heads=32, buckets=32, max_distance=128, ragged=False),
        # one token: a product of a vector with both weights, bound by reading them
        dict(name="ff_token", op="gated_ff", mode="infer", rows=1, dim=4096, hidden=10240, act="gelu_tanh"),
        # one prompt
        dict(name="ff_prompt", op="gated_ff", mode="infer", rows=226, dim=4096, hidden=10240, act="gelu_tanh"),
        # 64 prompts with 8-bit operands
        dict(name="ff_batch_e4m3", op="gated_ff", mode="e4m3", rows=14464, dim=4096, hidden=10240, act="gelu_tanh"),
        # a training step on 16 prompts: forward, then the gradients of the input and both weights
        dict(name="ff_train", op="gated_ff", mode="train", rows=3616, dim=4096, hidden=10240, act="gelu_tanh"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms_norm", "relbias_attn", "gated_ff"])
    if op == "rms_norm":
        return dict(op=op, mode=rng.choice(["infer", "e4m3", "train"]), rows=_log(rng, 1, 14464), dim=8 * _log(rng, 8, 1024),
                    stream=rng.choice(["float32", "bfloat16"]))
    if op == "relbias_attn":
        mode = rng.choice(["infer", "train"])
        length, heads, batch = _log(rng, 1, 4096), rng.randint(1, 64), _log(rng, 1, 32)
        room = 1.0e9 if mode == "infer" else 2.6e8            # the largest listed cases' pairs of positions
        heads = max(1, min(heads, int(room / length ** 2)))
        batch = max(1, min(batch, int(room / (length ** 2 * heads))))
        return dict(op=op, mode=mode, batch=batch, length=length, heads=heads, buckets=rng.choice([16, 32, 64]),
                    max_distance=rng.choice([64, 100, 128, 256]), ragged=rng.random() < 0.5)
    mode = rng.choice(["infer", "e4m3", "train"])
    rows = _log(rng, 1, 3616 if mode == "train" else 14464)
    return dict(op=op, mode=mode, rows=rows, dim=128 * _log(rng, 4, 32), hidden=32 * _log(rng, 16, 320), act=rng.choice(["gelu_tanh", "silu"]))


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _scale_of(rows):
    """The smallest power of two that brings a row's largest value to at most E4M3_MAX (never below 2^-126)."""
    m, e = torch.frexp(rows.abs().amax(dim=-1).clamp_min(2.0 ** -118))        # value = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    return torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126))


def _to_e4m3(rows):
    s = _scale_of(rows)
    return (rows / s[:, None]).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    state = dict(case)
    if case["op"] == "rms_norm":
        rows, dim = case["rows"], case["dim"]
        stream = getattr(torch, case["stream"])
        # a residual stream has a few channels that are far larger than the others
        channel = torch.exp(normal(dim, std=0.5)) * torch.where(torch.rand(dim, generator=g, device=dev) < 0.01, 20.0, 1.0)
        state.update(x=(normal(rows, dim) * channel).to(stream), delta=normal(rows, dim, std=0.5).to(torch.bfloat16),
                     w=0.2 + 0.05 * normal(dim), eps=1e-6)
        if case["mode"] == "train":
            state.update(dy=normal(rows, dim, std=1e-2).to(torch.bfloat16), dres=normal(rows, dim, std=1e-2).to(stream))
    elif case["op"] == "relbias_attn":
        B, S, H = case["batch"], case["length"], case["heads"]
        # q, k and v are the thirds of one projection's output, as the encoder has them
        qkv = normal(B, S, 3, H, 64)
        qkv[:, :, 0] *= 0.3
        qkv = qkv.to(torch.bfloat16)
        state.update(qkv=qkv, table=normal(case["buckets"], H, std=2.0).to(torch.bfloat16), mask=None)
        if case["ragged"]:                                    # lengths 0 ... S: a batch may hold an empty prompt
            lengths = torch.randint(0, S + 1, (B,), generator=g, device=dev)
            lengths[0] = S
            state["mask"] = torch.arange(S, device=dev)[None, :] < lengths[:, None]
        if case["mode"] == "train":
            state["do"] = normal(B, S, H, 64, std=1e-2).to(torch.bfloat16)
    else:
        rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
        x, wg, wu = normal(rows, dim), normal(hidden, dim, std=1.5 / math.sqrt(dim)), normal(hidden, dim, std=1.0 / math.sqrt(dim))
        if case["mode"] == "e4m3":
            for name, t in (("x", x), ("wg", wg), ("wu", wu)):
                state[name], state[name + "_scale"] = _to_e4m3(t)
        else:
            state.update(x=x.to(torch.bfloat16), wg=wg.to(torch.bfloat16), wu=wu.to(torch.bfloat16))
        if case["mode"] == "train":
            state["dh"] = normal(rows, hidden, std=1e-2).to(torch.bfloat16)
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    stream, w = s["x"].dtype, s["w"]
    h = s["x"].float() + s["delta"].float()
    r = torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + s["eps"])
    y = h * r * w
    if s["mode"] == "infer":
        return {"y": y.to(torch.bfloat16), "res": h.to(stream)}
    if s["mode"] == "e4m3":
        q, scale = _to_e4m3(y)
        return {"q": q, "scale": scale, "res": h.to(stream)}
    dy, xh = s["dy"].float(), h * r
    n = dy * w
    dx = r * (n - xh * (n * xh).mean(dim=-1, keepdim=True)) + s["dres"].float()
    return {"y": y.to(torch.bfloat16), "res": h.to(stream), "dx": dx.to(stream), "ddelta": dx.to(torch.bfloat16), "dw": (dy * xh).sum(dim=0)}


def _plain_buckets(S, num_buckets, max_distance, dev):
    """[S, S]: the bucket of key j seen from query i. Distances next to a bucket's border are computed in 64 bits."""
    at = torch.arange(S, device=dev)
    d = at[None, :] - at[:, None]
    half = num_buckets // 2
    near = half // 2
    n = d.abs()
    far = near + torch.floor(torch.log2(n.clamp_min(1).double() / near) / math.log2(max_distance / near) * (half - near) + 1e-9).long()
    return torch.where(n < near, n, far.clamp(max=half - 1)) + half * (d > 0)


def _plain_attn(s):
    q, k, v = (s["qkv"][:, :, i].float().transpose(1, 2).contiguous() for i in range(3))     # [B, H, S, 64]
    B, H, S, _ = q.shape
    bucket = _plain_buckets(S, s["buckets"], s["max_distance"], q.device)
    score = torch.matmul(q, k.transpose(2, 3).contiguous())
    score += s["table"].float().t()[:, bucket][None]
    if s["mask"] is not None:
        score.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
        v = v * s["mask"][:, None, :, None]
        k = k * s["mask"][:, None, :, None]
    top = score.amax(dim=-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    p /= p.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    out = {"o": torch.matmul(p, v).transpose(1, 2).to(torch.bfloat16)}
    if s["mode"] == "infer":
        return out
    do = s["do"].float().transpose(1, 2).contiguous()
    out["dv"] = torch.matmul(p.transpose(2, 3).contiguous(), do).transpose(1, 2).to(torch.bfloat16)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds -= (ds * p).sum(dim=-1, keepdim=True)
    ds *= p
    out["dq"] = torch.matmul(ds, k).transpose(1, 2).to(torch.bfloat16)
    out["dk"] = torch.matmul(ds.transpose(2, 3).contiguous(), q).transpose(1, 2).to(torch.bfloat16)
    hot = (bucket.reshape(1, -1) == torch.arange(s["buckets"], device=q.device)[:, None]).float()
    out["dtable"] = torch.matmul(hot, ds.sum(dim=0).reshape(H, S * S).t().contiguous()).to(torch.bfloat16)
    return out


def _plain_act(g, act):
    """The activation of g, and its derivative."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain_ff(s):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    if s["mode"] == "e4m3":
        x, wg, wu = x * s["x_scale"][:, None], wg * s["wg_scale"][:, None], wu * s["wu_scale"][:, None]
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    a, slope = _plain_act(g, s["act"])
    out = {"h": (a * u).to(torch.bfloat16)}
    if s["mode"] != "train":
        return out
    dh = s["dh"].float()
    dg, du = dh * u * slope, dh * a
    out["dx"] = (torch.matmul(dg, wg) + torch.matmul(du, wu)).to(torch.bfloat16)
    out["dwg"], out["dwu"] = torch.matmul(dg.t(), x).to(torch.bfloat16), torch.matmul(du.t(), x).to(torch.bfloat16)
    return out


# ---- the framework's calls -------------------------------------------------------------------------------------------------------------
def _own_norm(s):
    from aether_amd import ops
    if s["mode"] == "e4m3":
        q, scale, res = ops.rms_norm_e4m3(s["x"], s["w"], s["eps"], delta=s["delta"])
        return {"q": q, "scale": scale, "res": res}
    y, res = ops.rms_norm(s["x"], s["w"], s["eps"], delta=s["delta"])
    if s["mode"] == "infer":
        return {"y": y, "res": res}
    # a bf16 stream's stored sum is rounded, the norm's was not: both terms again
    h, delta = (s["x"], s["delta"]) if res.dtype == torch.bfloat16 else (res, None)
    dx, ddelta, dw = ops.rms_norm_backward(s["dy"], h, s["w"], s["eps"], dres=s["dres"], need_ddelta=True, delta=delta)
    return {"y": y, "res": res, "dx": dx, "ddelta": ddelta, "dw": dw}


def _own_attn(s):
    from aether_amd import ops
    q, k, v = s["qkv"].unbind(2)
    if s["mode"] == "infer":
        return {"o": ops.relbias_attn(q, k, v, s["table"], s["max_distance"], key_mask=s["mask"])}
    o, lse = ops.relbias_attn(q, k, v, s["table"], s["max_distance"], key_mask=s["mask"], need_lse=True)
    dq, dk, dv, dtable = ops.relbias_attn_backward(s["do"], q, k, v, o, lse, s["table"], s["max_distance"], key_mask=s["mask"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _own_ff(s):
    from aether_amd import ops
    if s["mode"] == "infer":
        return {"h": ops.gated_ff(s["x"], s["wg"], s["wu"], act=s["act"])}
    if s["mode"] == "e4m3":
        return {"h": ops.gated_ff_e4m3(s["x"], s["x_scale"], s["wg"], s["wg_scale"], s["wu"], s["wu_scale"], act=s["act"])}
    h, gu = ops.gated_ff(s["x"], s["wg"], s["wu"], act=s["act"], need_gu=True)
    dx, dwg, dwu = ops.gated_ff_backward(s["dh"], s["x"], s["wg"], s["wu"], gu, act=s["act"])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}


def run(state):
    if own:
        return {"rms_norm": _own_norm, "relbias_attn": _own_attn, "gated_ff": _own_ff}[state["op"]](state)
    return {"rms_norm": _plain_norm, "relbias_attn": _plain_attn, "gated_ff": _plain_ff}[state["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "rms_norm":
        rows, dim, wide = case["rows"], case["dim"], 4 if case["stream"] == "float32" else 2
        forward = rows * dim * (wide + 2 + wide + (1 if case["mode"] == "e4m3" else 2)) + 4 * dim + (4 * rows if case["mode"] == "e4m3" else 0)
        if case["mode"] != "train":
            return {"bytes": forward, "flops": 6 * rows * dim}
        return {"bytes": forward + rows * dim * (2 + wide + wide + wide + 2) + 8 * dim, "flops": 20 * rows * dim}
    if case["op"] == "relbias_attn":
        B, S, H = case["batch"], case["length"], case["heads"]
        kept = (1 + 0.5 * (B - 1)) / B if case["ragged"] else 1.0   # lengths are drawn from 0 ... S (the first is S): on average so many keys are left
        one, pairs = B * S * H * 64 * 2, B * H * S * S * kept
        table = 2 * case["buckets"] * H
        forward = one * (2 + 2 * kept) + table                      # q and o whole, k and v where a key counts
        if case["mode"] == "infer":
            return {"bytes": forward, "flops": 4 * 64 * pairs}
        # dO, o and q again, the keys that count again, three gradients; four more products of the scores' size
        return {"bytes": forward + one * (3 + 2 * kept) + 3 * one + 2 * table, "flops": (4 + 8) * 64 * pairs}
    rows, dim, hidden = case["rows"], case["dim"], case["hidden"]
    size = 1 if case["mode"] == "e4m3" else 2
    forward = size * (rows * dim + 2 * hidden * dim) + 2 * rows * hidden
    if case["mode"] != "train":
        return {"bytes": forward, "flops": 4 * rows * dim * hidden}
    return {"bytes": forward + 2 * (rows * hidden + 2 * rows * dim + 4 * hidden * dim), "flops": 12 * rows * dim * hidden}


# ---- 64 bits ------------------------------------------------------------------------------------------------------------------------------
def _exact_norm(s):
    x, w = (s["x"].double() + s["delta"].double()).requires_grad_(True), s["w"].double().requires_grad_(True)
    y = w * x / torch.sqrt(torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / x.shape[1] + s["eps"])
    if s["mode"] == "infer":
        return {"y": y.detach(), "res": x.detach()}
    if s["mode"] == "e4m3":
        y = y.detach()
        scale = torch.exp2(torch.ceil(torch.log2(torch.linalg.vector_norm(y, ord=math.inf, dim=1) / E4M3_MAX)))
        return {"q": y / scale[:, None], "scale": scale, "res": x.detach()}
    dx, dw = torch.autograd.grad((y * s["dy"].double()).sum() + (x * s["dres"].double()).sum(), (x, w))
    return {"y": y.detach(), "res": x.detach(), "dx": dx, "ddelta": dx, "dw": dw}


def _exact_borders(num_buckets, max_distance):
    """The distances at which the next bucket of one side begins, from whole numbers: bucket near + b begins at the smallest n with
    (n / near)^(half - near) >= (max_distance / near)^b."""
    half = num_buckets // 2
    near = half // 2
    found = list(range(1, near))
    for b in range(half - near):
        n = near
        while n ** (half - near) * near ** b < max_distance ** b * near ** (half - near):
            n += 1
        found.append(n)
    return found


def _exact_attn(s):
    leaf = [s["qkv"][:, :, i].double().requires_grad_(s["mode"] == "train") for i in range(3)]
    table = s["table"].double().requires_grad_(s["mode"] == "train")
    S, dev = leaf[0].shape[1], leaf[0].device
    borders = torch.tensor(_exact_borders(s["buckets"], s["max_distance"]), device=dev)
    rel = torch.arange(1 - S, S, device=dev)
    side = torch.searchsorted(borders, rel.abs(), right=True) + (rel > 0) * (s["buckets"] // 2)
    at = torch.arange(S, device=dev)
    bias = table[side][at[None, :] - at[:, None] + S - 1]                            # [S, S, H]
    q, k, v = (t.permute(0, 2, 1, 3) for t in leaf)
    score = torch.einsum("bhid,bhjd->bhij", q, k) + bias.permute(2, 0, 1)
    keep = None if s["mask"] is None else s["mask"][:, None, None, :]
    p = torch.softmax(score if keep is None else score.masked_fill(~keep, -1e30), dim=-1)
    p = p if keep is None else p * keep
    o = torch.einsum("bhij,bhjd->bihd", p, v)
    if s["mode"] == "infer":
        return {"o": o}
    dq, dk, dv, dtable = torch.autograd.grad((o * s["do"].double()).sum(), (*leaf, table))
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _exact_ff(s):
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    if s["mode"] == "e4m3":
        x, wg, wu = (t * s[n + "_scale"].double().unsqueeze(1) for t, n in ((x, "x"), (wg, "wg"), (wu, "wu")))
    leaf = [t.requires_grad_(s["mode"] == "train") for t in (x, wg, wu)]
    g, u = torch.einsum("md,fd->mf", leaf[0], leaf[1]), torch.einsum("md,fd->mf", leaf[0], leaf[2])
    h = u * (torch.nn.functional.silu(g) if s["act"] == "silu" else torch.nn.functional.gelu(g, approximate="tanh"))
    if s["mode"] != "train":
        return {"h": h}
    dx, dwg, dwu = torch.autograd.grad((h * s["dh"].double()).sum(), leaf)
    return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rms_norm": _exact_norm, "relbias_attn": _exact_attn, "gated_ff": _exact_ff}[case["op"]](s)
