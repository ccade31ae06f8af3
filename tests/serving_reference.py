"""Plain 64-bit restatements of the serving operators (rms-norm with 8-bit output, 4-bit-weight products, the 8-bit
paged cache and attention over it) and of how far a kernel with 32-bit sums may be from them."""

import numpy as np
import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype):
    """The largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


# ---- rms-norm ---------------------------------------------------------------------------------------

def rmsnorm(x, w, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, y if w is None else y * w.double()


def group_max(y, group):
    cols = y.shape[-1]
    wide = group or cols
    parts = torch.nn.functional.pad(y.abs(), (0, -(-cols // wide) * wide - cols)).reshape(y.shape[:-1] + (-1, wide))
    return parts.amax(-1)


def spread_scale(scale, cols, group):
    return scale.repeat_interleave(group or cols, -1)[..., :cols]


def check_held(got, scale, y, group, slack):
    """`got` (8-bit values) times `scale` against y: half a step of the 8-bit type, plus `slack` (relative) for the 32-bit arithmetic in front."""
    want = group_max(y, group) / TOP[got.dtype]
    assert ((scale.double() - want).abs() <= want * slack + 1e-45).all()
    s = spread_scale(scale.double(), y.shape[-1], group)
    if got.dtype == torch.int8:
        step = 0.5 * s
    else:  # e4m3: 2^-4 of the value, and half of the smallest step (2^-9) below 2^-6
        step = torch.maximum(y.abs() * 2.0**-4, s * 2.0**-10)
    off = (got.double() * s - y).abs()
    assert (off <= step + y.abs() * slack * 2).all(), (off - step).max()


# ---- products with 4-bit weights --------------------------------------------------------------------

def unpack(q):
    n, half = q.shape
    return torch.stack((q & 15, q >> 4), 2).reshape(n, half * 2)


def w4_weights(q, scales, zeros, group):
    of = torch.arange(q.shape[1] * 2) // group
    z = 8.0 if zeros is None else zeros.double()[:, of]
    return (unpack(q).double() - z) * scales.double()[:, of]


def w4_matmul(x, q, scales, zeros, bias, x_scale, group):
    """The product in 64 bits and the sum of the magnitudes that go into each of its elements."""
    x = x.double()
    if x_scale is not None:
        x = x * (x_scale.double() if x_scale.shape[-1] == 1 else x_scale.double().repeat_interleave(group, -1)[..., :x.shape[-1]])
    w = w4_weights(q, scales, zeros, group)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def w4_bound(y, size, k, dtype):
    """One rounding to the result's type, and a 32-bit sum: every x * (q - z) is exact, each of the K / 16 + 64 additions (16 products
    at a time, group sums times scales, partial sums, bias) is off by at most 2^-22 of the magnitudes summed so far."""
    out = 0.0 if dtype == torch.float32 else half_step(dtype)
    return y.abs() * out + size * (k / 16 + 64) * 2.0**-22 + (2.0**-25 if dtype == torch.float16 else 0.0)


# ---- the 8-bit paged cache --------------------------------------------------------------------------

def hold(x, dtype):
    x = np.asarray(x, dtype=np.float32)
    if dtype == torch.int8:
        x = np.clip(np.nan_to_num(np.rint(x), nan=0.0), -127, 127)
        return torch.from_numpy(x).to(torch.int8)
    return torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn)


def append(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, cu):
    """In place on CPU tensors, sequence by sequence and block by block, with the f32 arithmetic of the definition: a scale is the largest
    magnitude times 1 / Q, a held value the rounded quotient."""
    pages, heads, block, dim = k_cache.shape
    for b in range(len(lens)):
        n = int(cu[b + 1] - cu[b])
        start, length = int(lens[b]) - n, int(lens[b])
        for blk in range(max(start, 0) // block, -(-length // block)):
            lo, hi = max(start, blk * block), min(length, (blk + 1) * block)
            if lo < 0 or blk >= table.shape[1] or not 0 <= int(table[b, blk]) < pages or lo >= hi:
                continue
            page = int(table[b, blk])
            for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
                for h in range(heads):
                    new = x[int(cu[b]) + lo - start:int(cu[b]) + hi - start, h].float().numpy()
                    top = np.float32(TOP[cache.dtype])
                    before = np.float32(scale[page, h]) if lo > blk * block else np.float32(0)
                    after = np.maximum(before, np.abs(new).max() * (np.float32(1) / top))
                    div = after if after != 0 else np.float32(1)
                    with np.errstate(invalid="ignore", divide="ignore"):
                        if not after == before:
                            old = cache[page, h, :lo - blk * block].float().numpy()
                            cache[page, h, :lo - blk * block] = hold(old * before / div, cache.dtype)
                        cache[page, h, lo - blk * block:hi - blk * block] = hold(new / div, cache.dtype)
                    scale[page, h] = float(after)


def attention(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, window):
    """o, lse in 64 bits, and a bound on the error of a kernel that rounds the softmax's numerators once to 16 bits (2^-11 covers the
    rounding, 2^-18 the exponential) and whose scores have 32-bit sums; tokens outside every sequence are NaN."""
    pages, heads, block, dim = k_cache.shape
    o = torch.full(q.shape, float("nan"), dtype=torch.float64)
    lse = torch.full(q.shape[:2], float("nan"), dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(o), torch.zeros_like(lse)
    group = q.shape[1] // heads
    for b in range(len(lens)):
        n = int(cu[b + 1] - cu[b])
        for i in range(n):
            pos, t = int(lens[b]) - n + i, int(cu[b]) + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                o[t], lse[t] = 0.0, -float("inf")
                continue
            at = torch.arange(lo, pos + 1)
            blk = at // block
            if int(blk[-1]) >= table.shape[1] or not bool(((table[b, blk] >= 0) & (table[b, blk] < pages)).all()):
                continue
            page = table[b, blk].long()
            kk = k_cache[page, :, at % block].double() * k_scale[page].double()[:, :, None]
            vv = v_cache[page, :, at % block].double() * v_scale[page].double()[:, :, None]
            qq = q[t].double().reshape(heads, group, dim)
            s = torch.einsum("hgd,jhd->hgj", qq, kk) * scale
            size = (torch.einsum("hgd,jhd->hgj", qq.abs(), kk.abs()) * abs(scale)).amax(-1)
            p = torch.softmax(s, -1)
            o[t] = torch.einsum("hgj,jhd->hgd", p, vv).reshape(-1, dim)
            lse[t] = torch.logsumexp(s, -1).reshape(-1)
            wrong = size * (dim / 16 + 4) * 2.0**-22 + 2.0**-21  # of a score, in units of 1
            spread = torch.einsum("hgj,jhd->hgd", p, vv.abs())
            bound[t] = (spread * (2.0**-11 + 2.0**-18 + 2 * wrong[..., None])).reshape(-1, dim) + o[t].abs() * half_step(q.dtype)
            bound[t] += vv.abs().nan_to_num(nan=0.0).max() * 2.0**-24  # numerators below the 16-bit range, and results below f16's; a NaN counts for its own column
            lse_bound[t] = (wrong + 2.0**-20).reshape(-1) + lse[t].abs() * 2.0**-22
    return o, lse, bound, lse_bound
