"""Cases for the operators of a decoder layer's serving step: rms-norm with the residual's addition and
8-bit output, products with 4-bit weights, the 8-bit paged key/value cache's append, and attention over
that cache.  ``run`` computes a case with elementary torch operations in 32 bits, or, where ``own`` is
true, with this package's kernels; ``exact`` restates the definitions in 64 bits."""

import math

import torch

own = False

DEV = "cuda"
FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HELD = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
TOP = {"e4m3": 448.0, "i8": 127.0}
EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the norm in front of a product, one decoding step of 16 sequences: latency
        {"name": "norm_step", "op": "norm", "rows": 16, "cols": 4096, "type": "bf16", "out": "e4m3", "group": 0, "residual": True},
        # a ragged prompt chunk kept in 32 bits, no 8-bit output, width not a multiple of any tile
        {"name": "norm_f32_odd", "op": "norm", "rows": 1021, "cols": 5001, "type": "f32", "out": "same", "group": 0, "residual": True},
        # a large prefill batch, scales for each 128 columns
        {"name": "norm_prefill", "op": "norm", "rows": 16384, "cols": 8192, "type": "bf16", "out": "e4m3", "group": 128, "residual": True},
        # one token through a square projection: latency
        {"name": "w4_token", "op": "w4", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "group": 128, "zeros": False, "bias": False, "rowscale": False},
        # a short draft's tokens, small groups with zero points, odd number of rows and outputs
        {"name": "w4_draft", "op": "w4", "m": 7, "n": 5003, "k": 8192, "type": "f16", "group": 32, "zeros": True, "bias": True, "rowscale": False},
        # a decoding batch of 64 with 8-bit activations through a wide projection
        {"name": "w4_batch", "op": "w4", "m": 64, "n": 16384, "k": 8192, "type": "e4m3", "group": 128, "zeros": False, "bias": False, "rowscale": True},
        # one new token for each of 128 sequences: latency
        {"name": "append_step", "op": "append", "batch": 128, "new": 1, "ctx": 512, "heads": 8, "dim": 128, "block": 16, "type": "bf16", "held": "e4m3", "ragged": False},
        # prompt chunks of different lengths, int8, larger blocks
        {"name": "append_chunk", "op": "append", "batch": 6, "new": 8192, "ctx": 777, "heads": 8, "dim": 128, "block": 64, "type": "f16", "held": "i8", "ragged": True},
        # a single short conversation: latency
        {"name": "attn_short", "op": "attn", "batch": 1, "new": 1, "ctx": 701, "qheads": 32, "heads": 8, "dim": 128, "block": 16, "type": "bf16", "held": "e4m3", "window": 0, "ragged": False},
        # a decoding batch of mixed lengths
        {"name": "attn_batch", "op": "attn", "batch": 64, "new": 1, "ctx": 8192, "qheads": 32, "heads": 8, "dim": 128, "block": 16, "type": "bf16", "held": "e4m3", "window": 0, "ragged": False},
        # drafts of up to 5 tokens checked at once, narrow heads, a sliding window, int8
        {"name": "attn_draft", "op": "attn", "batch": 33, "new": 5, "ctx": 3001, "qheads": 16, "heads": 4, "dim": 64, "block": 32, "type": "f16", "held": "i8", "window": 2048, "ragged": True},
        # two very long documents, many query heads to a key head
        {"name": "attn_long", "op": "attn", "batch": 2, "new": 1, "ctx": 131072, "qheads": 64, "heads": 8, "dim": 128, "block": 64, "type": "bf16", "held": "e4m3", "window": 0, "ragged": False},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "w4", "append", "attn"])
    if op == "norm":
        held = rng.choice(["same", "e4m3", "e4m3"])
        group = rng.choice([0, 64, 128]) if held == "e4m3" else 0
        cols = _spread(rng, 256, 8192)
        cols = (cols + 127) // 128 * 128 if group else cols
        return {"op": op, "rows": min(_spread(rng, 1, 16384), (1 << (25 if held == "same" else 27)) // cols), "cols": cols, "type": rng.choice(["bf16", "f16", "f32"]) if held == "same" else rng.choice(["bf16", "f16"]),
                "out": held, "group": group, "residual": rng.random() < 0.7}
    if op == "w4":
        kind = rng.choice(["bf16", "f16", "e4m3"])
        return {"op": op, "m": _spread(rng, 1, 64), "n": _spread(rng, 512, 16384), "k": (_spread(rng, 512, 8192) + 31) // 32 * 32, "type": kind,
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "bias": rng.random() < 0.3, "rowscale": kind == "e4m3" and rng.random() < 0.5}
    heads = rng.choice([1, 2, 4, 8])
    d = {"op": op, "heads": heads, "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64]), "type": rng.choice(["bf16", "f16"]), "held": rng.choice(["e4m3", "i8"])}
    if op == "append":
        batch = _spread(rng, 1, 128)
        new = rng.choice([1, 1, 2, 5, _spread(rng, 8, 8192)])
        new = max(1, min(new, 32768 // batch))
        return {**d, "batch": batch, "new": new, "ctx": _spread(rng, 1, 1000), "ragged": new > 1 and rng.random() < 0.6}
    batch = _spread(rng, 1, 64)
    new = rng.choice([1, 1, 1, 2, 3, 5])
    return {**d, "batch": batch, "new": new, "ctx": _spread(rng, 16, max(32, 250000 // batch)), "qheads": heads * rng.choice([1, 3, 4, 8]),
            "window": rng.choice([0, 0, 1000]), "ragged": new > 1 and rng.random() < 0.5}


def _shares(n, top, low):
    """n whole numbers from `low` to `top`, spread evenly and in no order; the first is `top`."""
    return [max(low, int(round(top * (1.0 - (i * 0.6180339887498949) % 1.0)))) for i in range(n)]


def _lengths(case):
    """(new tokens, length with them) of every sequence: part of the case, the same for every seed.  `ctx` is
    what the longest one holds already."""
    new = _shares(case["batch"], case["new"], 1) if case["ragged"] else [case["new"]] * case["batch"]
    return new, [a + b for a, b in zip(_shares(case["batch"], case["ctx"], 0), new)]


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "i8": 1}
    if case["op"] == "norm":
        r, c, e = case["rows"], case["cols"], size[case["type"]]
        scales = 0 if case["out"] == "same" else r * (c // case["group"] if case["group"] else 1) * 4
        return {"bytes": r * c * (e * (3 if case["residual"] else 1) + (e if case["out"] == "same" else 1)) + c * e + scales, "flops": 6 * r * c}
    if case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        held = case["type"] == "e4m3"
        scales = n * groups * (2 + (1 if case["zeros"] else 0)) + (4 * m * (1 if case["rowscale"] else groups) if held else 0)
        return {"bytes": n * k // 2 + scales + m * k * size[case["type"]] + m * n * 2 + (n * 2 if case["bias"] else 0), "flops": 2 * m * n * k}
    new, lens = _lengths(case)
    if case["op"] == "append":
        values = 2 * sum(new) * case["heads"] * case["dim"]
        return {"bytes": values * (size[case["type"]] + 1), "flops": 3 * values}
    seen, read = 0, 0
    for n, length in zip(new, lens):
        spans = [(max(0, p - case["window"] + 1) if case["window"] else 0, p + 1) for p in range(length - n, length)]
        seen += sum(b - a for a, b in spans)
        read += spans[-1][1] - spans[0][0]
    cache = 2 * read * case["heads"] * case["dim"]
    return {"bytes": cache + cache // (case["block"] * case["dim"]) * 4 + 2 * sum(new) * case["qheads"] * case["dim"] * 2, "flops": 4 * seen * case["qheads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------

def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _hold(x, held, scale):
    """x / scale rounded to the 8-bit type."""
    y = x / scale
    return y.to(torch.float8_e4m3fn) if held == "e4m3" else torch.round(y).to(torch.int8)


def _cache(case, gen, blocks):
    """A cache filled block by block with normal values of varying size; (values, scales)."""
    shape = (blocks, case["heads"], case["block"], case["dim"])
    out, scales = torch.empty(shape, dtype=HELD[case["held"]], device=DEV), torch.empty(shape[:2], device=DEV)
    piece = max(1, (1 << 26) // math.prod(shape[1:]))
    for at in range(0, blocks, piece):
        x = _normal(gen, (min(piece, blocks - at),) + shape[1:]) * (0.5 + torch.rand((min(piece, blocks - at), shape[1], 1, 1), generator=gen, device=DEV))
        s = x.abs().amax((2, 3), keepdim=True) / TOP[case["held"]]
        out.view(torch.uint8)[at:at + piece] = _hold(x, case["held"], s).view(torch.uint8)
        scales[at:at + piece] = s[:, :, 0, 0]
    return out, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "norm":
        t, shape = FLOAT[case["type"]], (case["rows"], case["cols"])
        # activations have a few channels far larger than the rest
        size = torch.where(torch.rand(case["cols"], generator=gen, device=DEV) < 0.005, 20.0, 1.0)
        s["x"] = (_normal(gen, shape) * size).to(t)
        s["r"] = (_normal(gen, shape) * size * 2).to(t) if case["residual"] else None
        s["w"] = (1 + 0.2 * _normal(gen, (case["cols"],))).to(t)
    elif case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        held = case["type"] == "e4m3"
        s["out"] = torch.bfloat16 if held else FLOAT[case["type"]]
        s["q"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=DEV, dtype=torch.uint8)
        s["scales"] = (0.002 + 0.01 * torch.rand((n, groups), generator=gen, device=DEV)).to(s["out"])
        s["zeros"] = torch.randint(5, 11, (n, groups), generator=gen, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = _normal(gen, (n,), s["out"]) if case["bias"] else None
        x = _normal(gen, (m, k))
        if held:
            wide = k if case["rowscale"] else case["group"]
            x = torch.nn.functional.pad(x, (0, -(-k // wide) * wide - k)).view(m, -1, wide)
            xs = x.abs().amax(2, keepdim=True) / 448.0
            s["x"] = _hold(x, "e4m3", xs).view(m, -1)[:, :k].contiguous()
            s["xs"] = xs.view(m, -1).contiguous()
        else:
            s["x"], s["xs"] = x.to(s["out"]), None
    else:
        new, lens = _lengths(case)
        per = [-(-length // case["block"]) for length in lens]
        most, blocks = max(per), sum(per) + 3
        order = torch.randperm(blocks, generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
        count = torch.tensor(per, device=DEV)
        first = torch.cumsum(count, 0) - count
        at = torch.arange(most, device=DEV)[None]
        s["table"] = torch.where(at < count[:, None], order[(first[:, None] + at).clamp(max=blocks - 1)], 0).to(torch.int32)
        s["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        s["cu"] = torch.nn.functional.pad(torch.cumsum(torch.tensor(new, device=DEV), 0), (1, 0)).to(torch.int32) if case["ragged"] else None
        s["most_new"] = case["new"]
        s["kc"], s["ks"] = _cache(case, gen, blocks)
        s["vc"], s["vs"] = _cache(case, gen, blocks)
        t, total = FLOAT[case["type"]], sum(new)
        if case["op"] == "append":
            s["k"], s["v"] = (_normal(gen, (total, case["heads"], case["dim"]), t) for _ in range(2))
        else:
            s["q"] = _normal(gen, (total, case["qheads"], case["dim"]), t)
    return s


# ---- the plain forms ------------------------------------------------------------------------------

def _norm(s):
    case = s["case"]
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"].float()
    out = {"h": None if s["r"] is None else h.to(s["x"].dtype)}
    if case["out"] == "same":
        return {**out, "y": y.to(s["x"].dtype)}
    y = y.view(case["rows"], -1, case["group"] or case["cols"])
    scale = y.abs().amax(2, keepdim=True) / TOP[case["out"]]
    return {**out, "y": _hold(y, case["out"], scale).view(case["rows"], -1), "scale": scale.view(case["rows"], -1)}


def _w4(s):
    case = s["case"]
    n, k, g = case["n"], case["k"], case["group"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), 2).view(n, k).float()
    of = torch.arange(k, device=DEV) // g
    q = (q - (8.0 if s["zeros"] is None else s["zeros"].float()[:, of])) * s["scales"].float()[:, of]
    x = s["x"].float()
    if s["xs"] is not None:
        x = x * (s["xs"] if case["rowscale"] else s["xs"][:, of])
    y = x @ q.t()
    return {"y": (y if s["bias"] is None else y + s["bias"].float()).to(s["out"])}


def _append(s):
    case = s["case"]
    b, bs, total = s["lens"].numel(), case["block"], s["k"].shape[0]
    cu = torch.arange(b + 1, device=DEV, dtype=torch.int32) * (total // b) if s["cu"] is None else s["cu"]
    start = s["lens"] - (cu[1:] - cu[:-1])
    # the blocks that take new tokens: [sequence, block]; a sequence with fewer of them names its last one again
    blk = start[:, None] // bs + torch.arange((s["most_new"] + bs - 2) // bs + 1, device=DEV)[None]
    blk = torch.minimum(blk, (s["lens"] - 1)[:, None] // bs)
    page = s["table"].gather(1, blk.long()).long()
    pos = blk[:, :, None] * bs + torch.arange(bs, device=DEV)
    old = pos < start[:, None, None]
    fresh = ~old & (pos < s["lens"][:, None, None])
    token = torch.where(fresh, pos + (cu[:-1] - start)[:, None, None], 0).long()
    old, fresh = old[:, :, None, :, None], fresh[:, :, None, :, None]
    out = {}
    for x, c, sc in (("k", "kc", "ks"), ("v", "vc", "vs")):
        x = torch.where(fresh, s[x].float()[token].transpose(2, 3), 0.0)
        before = torch.where(old.any(3)[..., 0], s[sc][page], 0.0)
        after = torch.maximum(before, x.abs().amax((3, 4)) / TOP[case["held"]])
        wide = torch.where(after > 0, after, 1.0)[..., None, None]
        bits = s[c].view(torch.uint8)[page]
        again = _hold(bits.view(s[c].dtype).float() * before[..., None, None], case["held"], wide).view(torch.uint8)
        bits = torch.where(fresh, _hold(x, case["held"], wide).view(torch.uint8), torch.where(old & (after > before)[..., None, None], again, bits))
        s[c].view(torch.uint8)[page] = bits
        s[sc][page] = after
        out[c], out[sc] = s[c], s[sc]
    return out


def _attn(s):
    case = s["case"]
    b, h, d, bs = s["lens"].numel(), case["heads"], case["dim"], case["block"]
    total, group = s["q"].shape[0], case["qheads"] // h
    cu = torch.arange(b + 1, device=DEV, dtype=torch.int32) * (total // b) if s["cu"] is None else s["cu"]
    n = (cu[1:] - cu[:-1])[:, None]
    most = s["most_new"]
    at = torch.arange(most, device=DEV)[None]
    q = s["q"].float()[(cu[:-1, None] + at).clamp(max=total - 1).long()]
    q = q.view(b, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * group, d)
    page = s["table"].long()
    span = page.shape[1] * bs
    spread = lambda c, sc: (c.view(torch.uint8)[page].view(c.dtype).float() * sc[page][:, :, :, None, None]).transpose(1, 2).reshape(b, h, span, d)  # noqa: E731
    pos = (s["lens"][:, None] - n + at)[:, :, None]
    col = torch.arange(span, device=DEV)[None, None]
    seen = (col <= pos) & (col >= 0 if not case["window"] else col > pos - case["window"])
    seen = seen[:, None, :, None].expand(b, 1, most, group, span).reshape(b, 1, most * group, span)
    score = (q @ spread(s["kc"], s["ks"]).transpose(2, 3)) * (1.0 / math.sqrt(d))
    score = torch.where(seen, score, -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - top)
    total_p = p.sum(3, keepdim=True)
    held = spread(s["vc"], s["vs"])
    held = torch.where(seen.any(2)[..., None], held, 0.0)
    o = (p @ held) / total_p
    lse = (top + torch.log(total_p)).view(b, h, most, group)
    o = o.view(b, h, most, group, d)
    valid = at < n
    return {"o": o.permute(0, 2, 1, 3, 4)[valid].reshape(total, -1, d).to(s["q"].dtype), "lse": lse.permute(0, 2, 1, 3)[valid].reshape(total, -1)}


def run(s):
    case = s["case"]
    if own:
        from intent_ir_b200 import ops

        if case["op"] == "norm":
            y, scale, h = ops.rmsnorm(s["x"], s["w"], residual=s["r"], eps=EPS, out_dtype=None if case["out"] == "same" else HELD[case["out"]], group=case["group"])
            return {"h": h, "y": y} if scale is None else {"h": h, "y": y, "scale": scale}
        if case["op"] == "w4":
            return {"y": ops.w4_matmul(s["x"], s["q"], s["scales"], zeros=s["zeros"], bias=s["bias"], x_scale=s["xs"], group=case["group"], out_dtype=s["out"])}
        if case["op"] == "append":
            ops.kv8_append(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], cu_new=s["cu"])
            return {"kc": s["kc"], "ks": s["ks"], "vc": s["vc"], "vs": s["vs"]}
        o, lse = ops.attention_kv8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], cu_new=s["cu"], window=case["window"], return_lse=True)
        return {"o": o, "lse": lse}
    return {"norm": _norm, "w4": _w4, "append": _append, "attn": _attn}[case["op"]](s)


# ---- the definitions in 64 bits -------------------------------------------------------------------
# 8-bit values are given before their rounding: that is what the rounded ones stand for.

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        got = {"h": [], "y": [], "scale": []}
        for at in range(0, case["rows"], 2048):
            h = s["x"][at:at + 2048].double()
            if s["r"] is not None:
                h = h + s["r"][at:at + 2048].double()
            y = h / torch.sqrt(torch.sum(h ** 2, 1, keepdim=True) / case["cols"] + EPS) * s["w"].double()
            if case["out"] != "same":
                wide = case["group"] or case["cols"]
                parts = y.reshape(h.shape[0], case["cols"] // wide, wide)
                sc = torch.max(parts.abs(), 2).values / TOP[case["out"]]
                y = (parts / sc[:, :, None]).reshape(h.shape)
                got["scale"].append(sc)
            got["h"].append(h if s["r"] is not None else None)
            got["y"].append(y)
        out = {"h": None if s["r"] is None else torch.cat(got["h"]), "y": torch.cat(got["y"])}
        return {**out, "scale": torch.cat(got["scale"])} if got["scale"] else out
    if case["op"] == "w4":
        y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device=DEV)
        for g, at in enumerate(range(0, case["k"], case["group"])):
            end = min(case["k"], at + case["group"])
            byte = s["q"][:, at // 2:end // 2].to(torch.int64)
            q = torch.empty((case["n"], end - at), dtype=torch.float64, device=DEV)
            q[:, 0::2], q[:, 1::2] = (byte % 16).double(), (byte // 16).double()
            q -= 8.0 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
            x = s["x"][:, at:end].double()
            if s["xs"] is not None:
                x = x * s["xs"][:, 0 if case["rowscale"] else g][:, None].double()
            y += torch.mm(x, (q * s["scales"][:, g:g + 1].double()).t())
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    new, lens = _lengths(case)
    table, bs = s["table"].cpu().tolist(), case["block"]
    if case["op"] == "append":
        out = {"kc": s["kc"].double(), "ks": s["ks"].double(), "vc": s["vc"].double(), "vs": s["vs"].double()}
        for x, c, sc in (("k", "kc", "ks"), ("v", "vc", "vs")):
            start = 0
            for i, (n, length) in enumerate(zip(new, lens)):
                for at in range((length - n) // bs, -(-length // bs)):
                    lo, hi, page = max(length - n, at * bs), min(length, at * bs + bs), table[i][at]
                    fresh = s[x][start + lo - (length - n):start + hi - (length - n)].double().transpose(0, 1)
                    was = out[sc][page] if lo > at * bs else torch.zeros_like(out[sc][page])
                    now = torch.maximum(was, fresh.abs().amax((1, 2)) / TOP[case["held"]])
                    out[c][page][:, :lo - at * bs] *= (was / now)[:, None, None]
                    out[c][page][:, lo - at * bs:hi - at * bs] = fresh / now[:, None, None]
                    out[sc][page] = now
                start += n
        return out
    outs, lses, start, group = [], [], 0, case["qheads"] // case["heads"]
    for i, (n, length) in enumerate(zip(new, lens)):
        low = max(0, length - n - case["window"] + 1) // bs if case["window"] else 0
        pages = s["table"][i, low:-(-length // bs)].long()
        o = torch.empty((n, case["qheads"], case["dim"]), dtype=torch.float64, device=DEV)
        lse = torch.empty((n, case["qheads"]), dtype=torch.float64, device=DEV)
        for head in range(case["heads"]):
            k, v = ((c.view(torch.uint8)[pages, head].view(c.dtype).double() * sc[pages, head].double()[:, None, None]).reshape(-1, case["dim"])[:length - low * bs]
                    for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            for j in range(n):
                end = length - n + j + 1 - low * bs
                a = max(0, end - case["window"]) if case["window"] else 0
                at = slice(head * group, head * group + group)
                score = s["q"][start + j, at].double() @ k[a:end].t() / math.sqrt(case["dim"])
                lse[j, at] = torch.logsumexp(score, 1)
                o[j, at] = torch.softmax(score, 1) @ v[a:end]
        outs.append(o)
        lses.append(lse)
        start += n
    return {"o": torch.cat(outs), "lse": torch.cat(lses)}
