"""Definitions in 64 bits that the tests of the 8-bit cache and of sampling compare with."""
import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def scale_for(amax: float) -> float:
    """The smallest power of two s with amax <= 448 s, 2^-100 at least."""
    if amax == 0.0:
        return 2.0 ** -100
    s = 2.0 ** math.ceil(math.log2(amax / 448.0))
    while amax > 448.0 * s:
        s *= 2.0
    while amax <= 448.0 * (s / 2):
        s /= 2.0
    return max(s, 2.0 ** -100)


def to_code(x: torch.Tensor, s: float) -> torch.Tensor:
    """Codes of float64 values at scale s (what is not finite: NaN)."""
    y = torch.where(x.isfinite(), x / s, torch.full_like(x, math.nan))
    return y.float().to(E4M3)


def append(x, cache, scale, layer, slots):
    """Rows x (n, H, D) float64 into codes ``cache`` (L, NB, BS, H, D) and scales (L, NB, H), all on
    the CPU, in place."""
    _, NB, BS, H, _ = cache.shape
    by_block = {}
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < NB * BS:
            by_block.setdefault(s // BS, {})[s % BS] = r  # of equal slots the last one counts
    rows_of = {}
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < NB * BS:
            rows_of.setdefault(s // BS, []).append(r)
    for b, at in by_block.items():
        rows = x[rows_of[b]]
        for h in range(H):
            v = rows[:, h].abs()
            v = v[v.isfinite()]
            need = scale_for(float(v.max()) if v.numel() else 0.0)
            old = float(scale[layer, b, h])
            if not (0.0 < old < math.inf):
                old = 0.0
            new = need if 0 in at else max(need, old)
            if 0 not in at and new != old:
                for o in range(BS):
                    if o not in at:
                        held = cache[layer, b, o, h].double() * (old / new)
                        cache[layer, b, o, h] = held.float().to(E4M3)
            scale[layer, b, h] = new
            for o, r in at.items():
                cache[layer, b, o, h] = to_code(x[r, h], new)


def rotate(x, positions, inv_freq):
    """Rotate-half rotary of (n, heads, D) in float64."""
    ang = positions.double()[:, None] * inv_freq.double()[None]
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def attend(q, kc, vc, ks, vs, layer, tables, cu, ctx, scale):
    """Ragged causal attention in float64 over the CPU copies of an 8-bit cache.  Returns (out,
    sum of p|v| per output, largest |score| sum per row): the latter two bound rounding errors.
    Pages outside the pool do not take part; a row without any gives zeros."""
    n, hq, D = q.shape
    _, NB, BS, H, _ = kc.shape
    g = hq // H
    out = torch.zeros(n, hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    big = torch.zeros(n, hq, 1, dtype=torch.float64)
    for s in range(len(ctx)):
        lo, hi, c = int(cu[s]), int(cu[s + 1]), int(ctx[s])
        if hi == lo or c <= 0:
            continue
        ids = tables[s, :-(-c // BS)].long()
        good = (ids >= 0) & (ids < NB)
        safe = torch.where(good, ids, 0)
        k = (kc[layer, safe].double() * ks[layer, safe].double()[:, None, :, None]).flatten(0, 1)[:c]
        v = (vc[layer, safe].double() * vs[layer, safe].double()[:, None, :, None]).flatten(0, 1)[:c]
        ok = good.repeat_interleave(BS)[:c]
        pos = torch.arange(c - (hi - lo), c)
        seen = (torch.arange(c)[None] <= pos[:, None]) & ok[None]
        k = torch.where(ok[:, None, None], k, 0.0)
        v = torch.where(ok[:, None, None], v, 0.0)
        for h in range(hq):
            qq = q[lo:hi, h].double()
            sc = (qq @ k[:, h // g].T) * scale
            big[lo:hi, h, 0] = ((qq.abs() @ k[:, h // g].abs().T) * abs(scale)).masked_fill(~seen, 0).amax(-1)
            sc = sc.masked_fill(~seen, -math.inf)
            m = sc.amax(-1, keepdim=True)
            p = torch.where(seen, (sc - torch.where(m.isinf(), 0.0, m)).exp(), 0.0)
            z = p.sum(-1, keepdim=True)
            p = torch.where(z > 0, p / z, 0.0)
            # a masked position contributes nothing even where it holds NaN
            vv = v[:, h // g]
            used = seen.any(0)
            out[lo:hi, h] = p[:, used] @ vv[used]
            mag[lo:hi, h] = p[:, used] @ vv[used].abs()
    return out, mag, big


def attention_tolerance(dtype, out, mag, big, n_ctx, dim, p_bits):
    """Bound on |device - exact| per output: the output's own rounding; each weight p rounded to
    p_bits bits (and the 7.5e-5 of a polynomial exponential where p_bits is that of a tensor-core
    prefill); the score's fp32 sum of dim products, whose error moves p by a factor; the fp32 sum
    over the context."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    f32 = 2.0 ** -24
    weights = 2 * (2.0 ** -p_bits) + 2 * (2 * big + 4) * (dim + 8) * f32 + (n_ctx + 64) * f32
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    return half * out.abs() + weights * mag * (1 + half) + tiny


def sample_row(x: np.ndarray, t, k, p, m, u):
    """(token, log probability) of one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not np.isfinite(x).any() and not (x == np.inf).any():
        return -1, math.nan
    top = x.max()
    z = np.where(x == top, 0.0, (x - top) / (t or 1.0)) if np.isfinite(top) else np.where(x == top, 0.0, -np.inf)
    logs = math.log(np.exp(z).sum())
    order = np.lexsort((np.arange(len(z)), -x))
    if t == 0:
        return int(order[0]), -logs
    if 0 < k < len(z):
        order = order[:k]
    w = np.exp(z[order])
    if p < 1:
        before = np.cumsum(w) - w
        keep = before < p * w.sum()
        keep[0] = True
        order = order[keep]
    w = np.exp(z[order])
    keep = (w >= min(m, 1.0)) & (w > 0)
    order = np.sort(order[keep])
    c = np.cumsum(np.exp(z[order]))
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(order) - 1)
    return int(order[i]), float(z[order[i]] - logs)
