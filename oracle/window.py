"""Windowed attention with sinks in float64, forward and gradients, with the
error that the kernels' roundings allow for each element (test infrastructure).

Roundings counted, u = half a step of the 16-bit type relative to the value:
* the output, dq, dk, dv rounded once: u |result|;
* probabilities rounded before p . v and P^T . dO: u sum p |v| (independent errors
  may all point one way in a bound);
* dS as two 16-bit parts in its products: u^2 sum |dS| |k|;
* delta = dO . O from the unrounded O (as two parts): P (u^2 |O| + error of p . v) . |dO|;
* everything else in float32: sums of n terms n 2^-24 of the sum of absolute
  values; an exponent (a logit of up to 2^5 times log2 e, formed from float32 sums
  of the head size's terms) 2^-16 of p.
"""
from __future__ import annotations

import torch

SLACK = 2.0 ** -16


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def visible(i: torch.Tensor, j: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    """[len(i), len(j)]: whether position i sees position j (window 0: none)."""
    i, j = i[:, None], j[None, :]
    seen = j <= i
    if window:
        seen = seen & ((j > i - window) | (j < sinks))
    return seen


def attend(q, k, v, seen, scale):
    """q [n, d], k, v [t, d] float64, seen [n, t] -> (out, sum p |v|, p).  Tokens that a row does
    not see do not reach it, whatever they hold."""
    logits = torch.where(seen, (q @ torch.nan_to_num(k).T) * scale, -torch.inf)
    top = logits.amax(1, keepdim=True) if logits.shape[1] else logits.new_zeros(len(q), 1)
    p = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    p = torch.where(seen, p, 0.0)
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    clean = torch.nan_to_num(v)
    return p @ clean, p @ clean.abs(), p


def out_bound(out, spread, n, dtype, rounded_p=True):
    u = half_step(dtype)
    return u * out.abs() + ((u if rounded_p else 2.0 ** -16) + SLACK + n * 2.0 ** -23) * spread + \
        torch.finfo(dtype).smallest_normal * u * 2


def gradients(q, k, v, dout, seen, scale, dtype):
    """Of one head: (out, dq, dk, dv) and the bounds of their errors."""
    u, n = half_step(dtype), len(q)
    out, spread, p = attend(q, k, v, seen, scale)
    e_out = out_bound(out, spread, n, dtype)
    e_sum = e_out - (u - u * u) * out.abs()
    dp = dout @ v.T
    delta = (dout * out).sum(1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ dout
    f = SLACK + n * 2.0 ** -23
    size = dout.abs() @ v.abs().T + (dout.abs() * out.abs()).sum(1, keepdim=True)
    e_ds = (u * u + f) * ds.abs() + p * ((dout.abs() * e_sum).sum(1, keepdim=True) + f * size)
    tiny = torch.finfo(dtype).smallest_normal * u * 2
    e_dq = u * dq.abs() + scale * (e_ds + f * ds.abs()) @ k.abs() * (1 + u) + tiny
    e_dk = u * dk.abs() + scale * (e_ds + f * ds.abs()).T @ q.abs() * (1 + u) + tiny
    e_dv = u * dv.abs() + (u + 2 * f) * p.T @ dout.abs() + tiny
    return (out, dq, dk, dv), (e_out, e_dq, e_dk, e_dv), p


def slots_to_rows(kc, vc, table, ctx, block):
    """Cached keys and values [ctx, kv heads, dims] of one sequence, and which are there.
    kc [blocks, heads, dims / 8, block, 8], vc [blocks, heads, dims, block]."""
    t = torch.arange(ctx)
    blk = table.long()[t // block]
    held = (blk >= 0) & (blk < kc.shape[0])
    blk = torch.where(held, blk, 0)
    k = kc[blk, :, :, t % block].flatten(2)
    return k, vc[blk, :, :, t % block], held


def paged(q, starts, lens, tables, kc, vc, block, window, sinks, scale, rounded_p=True):
    """q [rows, heads, dims] float64 over a cache -> (out, bound) float64; rows of no
    sequence NaN.  dtype of the bound: that of the cache tensors."""
    heads, kvh = q.shape[1], kc.shape[1]
    out = torch.full(q.shape, torch.nan, dtype=torch.float64)
    bound = torch.full(q.shape, torch.nan, dtype=torch.float64)
    for s, ctx in enumerate(lens):
        a, b = int(starts[s]), int(starts[s + 1])
        if a == b:
            continue
        ctx = min(ctx, tables.shape[1] * block) if ctx > 0 else 0
        k, v, held = slots_to_rows(kc, vc, tables[s], ctx, block)
        i = torch.arange(lens[s] - (b - a), lens[s])
        seen = visible(i, torch.arange(ctx), window, sinks) & held[None, :]
        for h in range(heads):
            x = h // (heads // kvh)
            o, spread, _ = attend(q[a:b, h], k[:, x].double(), v[:, x].double(), seen, scale)
            out[a:b, h] = o
            bound[a:b, h] = out_bound(o, spread, ctx, kc.dtype, rounded_p)
    return out, bound


def dense(q, k, v, dout, lens, window, sinks, scale, dtype):
    """Packed sequences, float64 in and out: (out, dq, dk, dv) and their bounds; a
    gradient's bound sums those of the heads that share a key."""
    res = [torch.zeros_like(t) for t in (q, q, k, v)]
    bounds = [torch.zeros_like(t) for t in (q, q, k, v)]
    group = q.shape[1] // k.shape[1]
    at = 0
    for n in lens:
        r = slice(at, at + n)
        i = torch.arange(n)
        seen = visible(i, i, window, sinks)
        for h in range(q.shape[1]):
            x = h // group
            vals, errs, _ = gradients(q[r, h], k[r, x], v[r, x], dout[r, h], seen, scale, dtype)
            for dst, src in ((res, vals), (bounds, errs)):
                dst[0][r, h], dst[1][r, h] = src[0], src[1]
                dst[2][r, x] += src[2]
                dst[3][r, x] += src[3]
        at += n
    return res, bounds


def within(y: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor):
    """(all finite and within the bound, the worst ratio)."""
    d = (y.double().cpu() - ref).abs()
    ratio = torch.where(bound > 0, d / bound, d)
    worst = float(ratio.max()) if ratio.numel() else 0.0
    return bool(torch.isfinite(y).all()) and worst <= 1.0, worst
