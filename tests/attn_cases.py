"""Inputs and 64-bit references of the attention operators (numpy-free, torch
float64 on the inputs' device; nothing of the library is used)."""
from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def paged(lens, page, heads, dim, dtype, g, token_major=False, spare=3, fill=float("nan")):
    """A cache with the requests' tokens in pages of random order and `fill` in
    every place past a request's length.  lens: [(new, length)].  Returns
    (k, v, page_table, k_dense, v_dense): the last two per request
    [length, heads, dim]."""
    counts = [-(-n // page) for _, n in lens]
    total, width = sum(counts) + spare, max(max(counts), 1) + 1
    order = torch.randperm(total, device="cuda", generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    shape = (total, page, heads, dim) if token_major else (total, heads, page, dim)
    k, v = (torch.full(shape, fill, dtype=dtype, device="cuda") for _ in range(2))
    ks, vs, at = [], [], 0
    for b, (_, n) in enumerate(lens):
        ks.append(normal(g, (n, heads, dim), dtype, 1.3))
        vs.append(normal(g, (n, heads, dim), dtype))
        for j in range(counts[b]):
            pg = order[at]
            at += 1
            table[b, j] = pg
            rows = min(page, n - j * page)
            for cache, src in ((k, ks[-1]), (v, vs[-1])):
                piece = src[j * page:j * page + rows]
                if token_major:
                    cache[pg, :rows] = piece
                else:
                    cache[pg, :, :rows] = piece.transpose(0, 1)
    return k, v, table.cuda(), ks, vs


def offsets_of(lens):
    out = [0]
    for n, _ in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda"), torch.tensor([n for _, n in lens], dtype=torch.int32,
                                                                            device="cuda")


def visible_mask(new, length, causal, window):
    """[new, length] truth values: which positions each new token sees."""
    p = torch.arange(length - new, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")[None]
    seen = torch.ones((new, length), dtype=torch.bool, device="cuda")
    if causal:
        seen &= j <= p
        if window:
            seen &= j > p - window
    elif window:
        seen &= (j - p).abs() < window
    return seen


def attention_ref(q, lens, ks, vs, scale, causal, window):
    """(out, lse, tol_of_out, tol_of_lse) in float64, over all rows of q.

    tol_of_out bounds the error of a computation that rounds the
    probabilities exp(s - max) to the 16-bit type before the product with V,
    sums them before that rounding, and rounds the result once:
      u sum(p |v|) + u |out|, p the normalised probabilities, u the type's
      unit roundoff; f16 adds 2^-25 sum|v| / sum exp(s - max) for
      probabilities below its normal range;
      fp32 scores: a head_dim-term dot product of relative error at most
      head_dim 2^-24 of scale sum|q k|, which scales every p by up to twice
      that; and the accumulation of n fp32 terms, n 2^-24 (blocked sums stay
      far below) -- both against sum(p |v|)."""
    u = UNIT[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    tol_lse = torch.zeros_like(lse)
    t = 0
    for b, (new, length) in enumerate(lens):
        if new and length:
            seen = visible_mask(new, length, causal, window)
            group = q.shape[1] // ks[b].shape[1]
            for h in range(q.shape[1]):
                qq = q[t:t + new, h].double()
                k, v = ks[b][:, h // group].double(), vs[b][:, h // group].double()
                s = (qq @ k.T * scale).masked_fill(~seen, -math.inf)
                size = (qq.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                top = s.amax(-1, keepdim=True).clamp(min=-1e300)
                e = torch.exp(s - top)
                total = e.sum(-1, keepdim=True)
                ok = total[:, 0] > 0
                p = e / total.clamp(min=1e-300)
                y, a = p @ v, p @ v.abs()
                score_err = 2 * q.shape[2] * 2.0 ** -24 * size + length * 2.0 ** -24
                bound = u * a + u * y.abs() + (2 * score_err + 2.0 ** -20) * a + 1e-30
                if q.dtype == torch.float16:
                    bound += 2.0 ** -25 * (seen.double() @ v.abs()) / total.clamp(min=1.0) + 2.0 ** -25
                out[t:t + new, h], tol[t:t + new, h] = y, bound
                z = (top + total.log())[:, 0]
                lse[t:t + new, h] = torch.where(ok, z, torch.full_like(z, -math.inf))
                tol_lse[t:t + new, h] = score_err[:, 0] + 2.0 ** -21 + 2.0 ** -22 * z.abs().clamp(max=1e30)
        t += new
    return out, lse, tol, tol_lse


def heads_ref(x, weight, eps, freq, amplitude, layout, where):
    """(y, tolerance): norm and rotation of [tokens, heads, dim] in float64.
    where: positions [tokens, pairs] or None.  The tolerance: one rounding to
    the type, and for the fp32 steps before it (sum of squares of dim terms,
    reciprocal root, three products and a sum; cos and sin to 2^-22 absolute,
    the angle's own fp32 form 2^-23 turns) 16 units of 2^-24 a term plus
    (|a| + |b|) amplitude 2^-19."""
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    slack = 24 * 2.0 ** -24 * y.abs()
    if freq is not None:
        n = freq.numel()
        a_at = torch.arange(n, device=x.device) * (1 if layout == "half" else 2)
        b_at = a_at + (n if layout == "half" else 1)
        t = where.double() * freq.double()
        cos, sin = (torch.cos(t) * amplitude)[:, None], (torch.sin(t) * amplitude)[:, None]
        a, b = y[..., a_at].clone(), y[..., b_at].clone()
        y[..., a_at], y[..., b_at] = a * cos - b * sin, b * cos + a * sin
        both = (a.abs() + b.abs()) * abs(amplitude)
        slack[..., a_at] = both * 2.0 ** -19
        slack[..., b_at] = both * 2.0 ** -19
    tol = UNIT[x.dtype] * y.abs() * (1 + 2.0 ** -8) + 2 * slack + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)
    return y, tol


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst error {float(err.max()):.3e}"
