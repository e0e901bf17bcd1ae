"""The operators of a text tower's layer, measured: RMS norm with residual and 8-bit output, dense layers on 4-bit weights with group scales, and
attention with a sliding window and always-visible first tokens. `run` computes them in their plain form, or with `own` through the package."""
import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1}


def listed():
    return [
        # a query's or memory's one new token through the norm ahead of an 8-bit dense layer: latency is all there is
        dict(name="norm_token", op="norm", rows=1, dim=384, dtype="bf16", residual=True, quant="int8", group=0, y=False),
        # a batch of texts of a tower with an odd width, in f32, with both outputs
        dict(name="norm_odd", op="norm", rows=1001, dim=771, dtype="f32", residual=False, quant="e4m3", group=64, y=True),
        # bulk ingest: every token of a large batch, residual added on the way
        dict(name="norm_batch", op="norm", rows=32768, dim=4096, dtype="bf16", residual=True, quant="e4m3", group=128, y=False),
        # one token through the q|k|v projection of a small encoder
        dict(name="w4_token_small", op="w4", rows=1, n=1152, k=384, group=32, zeros=False, dtype="bf16"),
        # odd sizes in f32: a pruned layer, a handful of tokens
        dict(name="w4_odd", op="w4", rows=5, n=1001, k=1234, group=64, zeros=True, dtype="f32"),
        # one token through the up projection of a large tower
        dict(name="w4_token", op="w4", rows=1, n=14336, k=4096, group=128, zeros=True, dtype="f16"),
        # sixteen callers' tokens, activations in 8 bits as the norm writes them
        dict(name="w4_int8_rows", op="w4", rows=16, n=4096, k=4096, group=128, zeros=False, dtype="int8"),
        # a short text's tokens through the widest layer
        dict(name="w4_text", op="w4", rows=64, n=28672, k=4096, group=128, zeros=False, dtype="bf16"),
        # a batch of texts in the encoder's own head layout (q|k|v of a token side by side), windowed both ways, first token visible to all
        dict(name="attn_texts", op="attn", seqs=96, lq=0, lmin=0, lmax=512, heads=12, kv_heads=12, dim=32, left=64, right=64, sinks=1, dtype="bf16"),
        # one token at the end of one long conversation
        dict(name="attn_token", op="attn", seqs=1, lq=1, lmin=32768, lmax=32768, heads=16, kv_heads=4, dim=64, left=4095, right=0, sinks=4, dtype="f16"),
        # a step of many conversations of all lengths, grouped heads
        dict(name="attn_tokens", op="attn", seqs=48, lq=1, lmin=0, lmax=32768, heads=32, kv_heads=8, dim=128, left=16383, right=0, sinks=4, dtype="bf16"),
        # a long document read at once
        dict(name="attn_document", op="attn", seqs=1, lq=0, lmin=8192, lmax=8192, heads=32, kv_heads=8, dim=128, left=2047, right=0, sinks=4, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo .. hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("norm", "w4", "attn"))
    if op == "norm":
        dim = _spread(rng, 64, 8192)
        rows = _spread(rng, 1, min(32768, 32768 * 4096 // dim))
        quant = rng.choice(("", "int8", "e4m3"))
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(("f32", "f16", "bf16")), residual=rng.random() < 0.6, quant=quant,
                    group=rng.choice((0, 32, 64, 128)), y=not quant or rng.random() < 0.3)
    if op == "w4":
        return dict(op=op, rows=_spread(rng, 1, 64), n=_spread(rng, 128, 16384), k=_spread(rng, 128, 7168), group=rng.choice((32, 64, 128)),
                    zeros=rng.random() < 0.5, dtype=rng.choice(("f32", "f16", "bf16", "int8")))
    dim, (heads, kv) = rng.choice((32, 64, 128)), rng.choice(((12, 12), (16, 4), (32, 8), (8, 1)))
    kind = rng.choice(("texts", "token", "document"))
    c = dict(op=op, seqs=1, lq=0, lmin=0, lmax=0, heads=heads, kv_heads=kv, dim=dim, left=_spread(rng, 16, 4096), right=0, sinks=rng.choice((0, 1, 4, 5)),
             dtype=rng.choice(("f16", "bf16")))
    if kind == "texts":
        c.update(seqs=_spread(rng, 1, 64), lmax=_spread(rng, 8, 512), left=_spread(rng, 8, 256), right=_spread(rng, 8, 256))
    elif kind == "token":
        c.update(seqs=_spread(rng, 1, 48), lq=rng.choice((1, 1, 1, 2, 5)), lmax=_spread(rng, 64, 32768))
    else:
        n = _spread(rng, 300, 6000)
        c.update(lmin=n, lmax=n)
    return c


def _lengths(c):
    """New tokens and keys of each sequence: the case's own, whatever the seed."""
    r = random.Random(1009 * c["seqs"] + 31 * c["lmax"] + c["lq"])
    if c["lmin"] == c["lmax"]:
        keys = [c["lmax"]] * c["seqs"]
    else:       # over the whole range, the longest one among them; an empty one where there is room
        keys = [min(c["lmax"], max(c["lmin"], int(math.exp(r.uniform(0, math.log(c["lmax"] + 0.99)))))) for _ in range(c["seqs"])]
        keys[0] = c["lmax"]
        if c["seqs"] > 4:
            keys[2] = c["lmin"]
    return [c["lq"] or n for n in keys], keys


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _quantized(w, group, zeros, g):
    """4-bit weights of a float matrix, two to a byte (the even one low), scales per group in f16 values, zero points."""
    n, k = w.shape
    ng = -(-k // group)
    p = torch.nn.functional.pad(w, (0, ng * group - k)).view(n, ng, group)
    if zeros:
        lo, hi = p.amin(2).clamp(max=0), p.amax(2).clamp(min=0)
        scale = ((hi - lo) / 15).clamp(min=1e-4).half().float()
        z = torch.round(-lo / scale).clamp(0, 15)
    else:
        scale = (p.abs().amax(2) / 7).clamp(min=1e-4).half().float()
        z = torch.full_like(scale, 8.0)
    q = (torch.round(p / scale[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :k]
    q = torch.nn.functional.pad(q, (0, k % 2))
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale.contiguous(), z.to(torch.uint8) if zeros else None


def _inputs(c, seed):
    g = _generator(seed)
    if c["op"] == "norm":
        t = TYPES[c["dtype"]]
        channel = torch.exp(0.5 * _normal(g, c["dim"]))          # some channels carry far more than others
        s = {"x": (_normal(g, c["rows"], c["dim"]) * channel).to(t), "weight": (1 + 0.2 * _normal(g, c["dim"])).to(t)}
        s["residual"] = (4 * _normal(g, c["rows"], c["dim"]) * channel).to(t) if c["residual"] else None
        return s
    if c["op"] == "w4":
        q, scale, z = _quantized(0.02 * _normal(g, c["n"], c["k"]), c["group"], c["zeros"], g)
        x = _normal(g, c["rows"], c["k"])
        s = {"q": q, "scale": scale, "zeros": z, "bias": 0.1 * _normal(g, c["n"]), "x_scale": None}
        if c["dtype"] == "int8":
            s["x_scale"] = x.abs().amax(1) / 127
            s["x"] = torch.round(x / s["x_scale"][:, None]).to(torch.int8)
        else:
            s["x"] = x.to(TYPES[c["dtype"]])
        return s
    t = TYPES[c["dtype"]]
    nq, nk = _lengths(c)
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    s = {"cu": torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=DEV), "kv_start": None, "kv_len": None}
    if c["lq"] == 0:            # self-attention: q|k|v of a token side by side, as the projection writes them
        qkv = _normal(g, sum(nq), heads + 2 * kv, d).to(t)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:                       # new tokens at the end of a cache: each sequence's keys have a place of their own in it, with room behind them
        start = [sum(nk[:i]) + 16 * i for i in range(len(nk))]
        total = start[-1] + nk[-1] + 16
        s["q"] = _normal(g, sum(nq), heads, d).to(t)
        s["k"], s["v"] = _normal(g, total, kv, d).to(t), _normal(g, total, kv, d).to(t)
        s["kv_start"] = torch.tensor(start, dtype=torch.int64, device=DEV)
        s["kv_len"] = torch.tensor(nk, dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "attn":
        s["longest"] = [max(v) for v in _lengths(case)]
    if own and case["op"] == "w4":      # weights are laid out once, when a program loads them
        from shodh_memory_amd import layers
        s["w4"] = layers.W4Weight.from_quantized(s["q"], s["scale"], s["zeros"], k=case["k"], group=case["group"])
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------------

def _norm_plain(s, c):
    h = s["x"].float()
    if c["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
    out = {"sum": h.to(s["x"].dtype) if c["residual"] else None, "y": y.to(s["x"].dtype) if c["y"] else None}
    if c["quant"]:
        top, dim, group = 127.0 if c["quant"] == "int8" else 448.0, c["dim"], c["group"] or c["dim"]
        ng = -(-dim // group)
        p = torch.nn.functional.pad(y, (0, ng * group - dim)).view(-1, ng, group)
        amax = p.abs().amax(2, keepdim=True)
        scale = amax / top
        v = (p * torch.where(amax > 0, top / amax, 0.0)).view(-1, ng * group)[:, :dim]
        out["scale"] = scale.view(-1, ng)
        q = torch.round(v).clamp(-127, 127).to(torch.int8) if c["quant"] == "int8" else v.clamp(-448, 448).to(torch.float8_e4m3fn)
        out["q"] = _values(q, out["scale"], c, s["x"].dtype)
    return out


def _values(q, scale, c, dtype):
    """What is held in 8 bits as numbers: e4m3 is a type of its own and goes out as it is, next to its scales; int8 as the values it stands for."""
    if c["quant"] == "e4m3":
        return q
    each = scale if scale.shape[1] == 1 else scale.repeat_interleave(c["group"], 1)[:, :c["dim"]]
    return (q * each).to(torch.float16 if dtype == torch.float32 else dtype)


def _w4_plain(s, c):
    q = torch.stack((s["q"] & 15, s["q"] >> 4), 2).view(c["n"], -1)[:, :c["k"]].float()
    each = torch.arange(c["k"], device=q.device) // c["group"]
    z = s["zeros"].float()[:, each] if c["zeros"] else 8.0
    w = (q - z) * s["scale"][:, each]
    y = s["x"].float() @ w.t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None]
    return (y + s["bias"]).to(torch.bfloat16 if c["dtype"] == "int8" else s["x"].dtype)


def _attn_plain(s, c):
    cu, (mq, mk) = s["cu"].long(), s["longest"]
    nq = cu[1:] - cu[:-1]
    start, nk = (cu[:-1], nq) if s["kv_start"] is None else (s["kv_start"], s["kv_len"].long())
    b, heads, kv, d = nq.numel(), c["heads"], c["kv_heads"], c["dim"]
    i, j = torch.arange(mq, device=cu.device), torch.arange(mk, device=cu.device)
    iq = torch.where(i < nq[:, None], cu[:-1, None] + i, 0)
    ik = torch.where(j < nk[:, None], start[:, None] + j, 0)
    q = s["q"].float()[iq].view(b, mq, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    k = s["k"][ik].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][ik].float().permute(0, 2, 1, 3).contiguous()
    p = (i[None, :] + (nk - nq)[:, None])[:, :, None]
    seen = (j < nk[:, None, None]) & (i[:, None] < nq[:, None, None])
    if c["right"] >= 0:
        seen = seen & (j <= p + c["right"])
    if c["left"] >= 0:
        seen = seen & ((j >= p - c["left"]) | (j < c["sinks"]))
    w = (q @ k).mul_(1.0 / math.sqrt(d)).view(b, kv, heads // kv, mq, mk).masked_fill_(~seen[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    w = w.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(b, kv, -1, mk) @ v).view(b, kv, heads // kv, mq, d) / torch.where(total > 0, total, 1.0)
    at = (torch.arange(b, device=cu.device)[:, None].expand(b, mq)[i < nq[:, None]], i.expand(b, mq)[i < nq[:, None]])
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, heads, d)[at]
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, mq, heads)[at]
    return {"out": o.to(s["q"].dtype), "lse": lse}


def run(state):
    c = state["case"]
    if not own:
        return {"norm": _norm_plain, "w4": _w4_plain, "attn": _attn_plain}[c["op"]](state, c)
    from shodh_memory_amd import layers
    if c["op"] == "norm":
        r = layers.rms_norm(state["x"], state["weight"], eps=1e-6, residual=state["residual"], want_y=c["y"], quant=c["quant"] or None, group=c["group"])
        out = {"sum": r.sum, "y": r.y}
        if c["quant"]:
            out["scale"] = r.scale
            out["q"] = _values(r.q, r.scale, c, state["x"].dtype)
        return out
    if c["op"] == "w4":
        return state["w4"].dense(state["x"], x_scale=state["x_scale"], bias=state["bias"], out_dtype=torch.bfloat16 if c["dtype"] == "int8" else None)
    o, lse = layers.window_attention(state["q"], state["k"], state["v"], state["cu"], left=c["left"], right=c["right"], sinks=c["sinks"],
                                     kv_start=state["kv_start"], kv_len=state["kv_len"], return_lse=True)
    return {"out": o, "lse": lse}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "norm":
        n, b = c["rows"] * c["dim"], BYTES[c["dtype"]]
        ng = -(-c["dim"] // (c["group"] or c["dim"]))
        held = n * (b + (2 * b if c["residual"] else 0) + (b if c["y"] else 0) + (1 if c["quant"] else 0))
        return {"bytes": held + c["dim"] * b + (4 * c["rows"] * ng if c["quant"] else 0), "flops": 8 * n}
    if c["op"] == "w4":
        ng = -(-c["k"] // c["group"])
        weights = c["n"] * (-(-c["k"] // 2)) + c["n"] * ng * 2 + (c["n"] * ng if c["zeros"] else 0)
        return {"bytes": weights + c["rows"] * (c["k"] * BYTES[c["dtype"]] + c["n"] * {"f32": 4}.get(c["dtype"], 2)) + 4 * c["n"],
                "flops": 2 * c["rows"] * c["n"] * c["k"]}
    pairs = keys = rows = 0
    for nq, nk in zip(*_lengths(c)):
        rows += nq
        first, lowest = nk, nk
        for i in range(nq):
            p = i + nk - nq
            hi = min(nk, p + c["right"] + 1) if c["right"] >= 0 else nk
            lo = max(0, p - c["left"]) if c["left"] >= 0 else 0
            if hi > 0:
                pairs += max(0, hi - lo) + min(c["sinks"], lo, hi)
                lowest = min(lowest, lo)
        if nq:
            keys += nk - lowest + min(c["sinks"], lowest)
    return {"bytes": 4 * rows * c["heads"] * c["dim"] + 4 * keys * c["kv_heads"] * c["dim"] + 4 * rows * c["heads"], "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if c["residual"] else 0)
        y = s["weight"].double() * h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / c["dim"] + 1e-6)
        out = {"sum": h if c["residual"] else None, "y": y if c["y"] else None}
        if c["quant"]:      # int8: the values that the rounded numbers stand for; e4m3: the numbers before they are rounded, in units of the scale next to them
            group = c["group"] or c["dim"]
            scale = torch.stack([part.abs().max(1).values for part in y.split(group, 1)], 1) / (127 if c["quant"] == "int8" else 448)
            out["scale"] = scale
            each = scale.repeat_interleave(group, 1)[:, :c["dim"]]
            v = y / each.clamp(min=1e-300)
            out["q"] = torch.round(v) * each if c["quant"] == "int8" else v
        return out
    if c["op"] == "w4":
        y = torch.zeros(c["rows"], c["n"], dtype=torch.float64, device=DEV)
        for g in range(-(-c["k"] // c["group"])):
            at = torch.arange(g * c["group"], min(c["k"], (g + 1) * c["group"]), device=DEV)
            q = (s["q"][:, at // 2] >> (4 * (at % 2)).to(torch.uint8)) & 15
            q = q.double() - (s["zeros"][:, g:g + 1].double() if c["zeros"] else 8)
            y += (s["x"][:, at].double() @ q.t().contiguous()) * s["scale"][:, g].double()
        return y * (s["x_scale"].double()[:, None] if s["x_scale"] is not None else 1) + s["bias"].double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
    at = 0
    for b, (nq, nk) in enumerate(zip(*_lengths(c))):
        first = at if s["kv_start"] is None else int(s["kv_start"][b])
        for i0 in range(0, nq, 2048):
            i1 = min(nq, i0 + 2048)
            pos = torch.arange(i0, i1, device=DEV)[:, None] + nk - nq
            j = torch.arange(nk, device=DEV)[None]
            hidden = (j > pos + c["right"]) if c["right"] >= 0 else torch.zeros_like(j + pos, dtype=torch.bool)
            if c["left"] >= 0:
                hidden = hidden | ((j < pos - c["left"]) & (j >= c["sinks"]))
            for h in range(c["heads"]):
                hk = h * c["kv_heads"] // c["heads"]
                score = s["q"][at + i0:at + i1, h].double() @ s["k"][first:first + nk, hk].double().t().contiguous() * c["dim"] ** -0.5
                score = score.masked_fill(hidden, float("-inf"))
                l = torch.logsumexp(score, 1)
                lse[at + i0:at + i1, h] = l
                w = torch.exp(score - torch.where(torch.isinf(l), 0.0, l)[:, None])
                out[at + i0:at + i1, h] = w @ s["v"][first:first + nk, hk].double()
        at += nq
    return {"out": out, "lse": lse}
