"""The 8-bit paged KV cache in 64 bits, token by token.

Caches are dicts of float64 tensors ``k``, ``v`` [P, Hkv, page, D] (the codes'
own values) and int64 exponents ``k_exp``, ``v_exp`` [P, Hkv, page / block]
(scale = 2^exp); -127 is the exponent of a zero byte.
"""
from __future__ import annotations

import math

import torch

E_MIN, E_MAX = -117, 119


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to even, saturated at 448; not finite -> NaN."""
    a = y.abs().clamp(max=448.0)
    ex = torch.floor(torch.log2(torch.clamp(a, min=2.0 ** -6)))
    step = torch.exp2(ex - 3)
    r = torch.copysign(torch.round(a / step) * step, y)  # torch.round: ties to even
    return torch.where(torch.isfinite(y), r, torch.full_like(r, math.nan))


def need_exp(amax: float) -> int:
    """The least e in [E_MIN, E_MAX] with amax <= 448 * 2^e."""
    e = E_MIN
    if amax > 0:
        m, ex = math.frexp(amax)  # m * 2^ex, m in [0.5, 1): 448 = 0.875 * 2^9
        e = ex - 9 + (1 if m > 0.875 else 0)
    return min(max(e, E_MIN), E_MAX)


def empty(P, Hkv, page, block, D=128):
    c = {n: torch.zeros(P, Hkv, page, D, dtype=torch.float64) for n in ("k", "v")}
    c.update({n + "_exp": torch.full((P, Hkv, page // block), -127, dtype=torch.int64) for n in ("k", "v")})
    return c


def from_bytes(k, v, k_scale, v_scale):
    """The oracle's cache of a cache's own tensors."""
    c = {"k": k.cpu().double(), "v": v.cpu().double()}
    c["k_exp"], c["v_exp"] = (s.cpu().view(torch.uint8).long() - 127 for s in (k_scale, v_scale))
    return c


def append(cache, k, v, slots):
    """The cache after one call with k, v [N, Hkv, D] (float64) at slots [N]."""
    P, H, page, _ = cache["k"].shape
    block = page // cache["k_exp"].shape[2]
    out = {n: t.clone() for n, t in cache.items()}
    blocks: dict = {}
    for n, s in enumerate(int(s) for s in slots):
        if 0 <= s < P * page:
            blocks.setdefault(s // block, {})[s % block] = n  # the last of a slot counts
    per = page // block
    for blk, members in blocks.items():
        pg, nb = divmod(blk, per)
        tok = list(members.values())
        for name, x in (("k", k), ("v", v)):
            for h in range(H):
                new = x[tok, h]
                fin = torch.where(torch.isfinite(new), new.abs(), torch.zeros_like(new))
                e = need_exp(float(fin.max()))
                old = int(out[name + "_exp"][pg, h, nb])
                anew = 0 in members
                if not anew:
                    e = max(e, old)
                rows = out[name][pg, h, nb * block:(nb + 1) * block]
                if anew:
                    rows.zero_()
                elif e != old:
                    rows.copy_(round_e4m3(rows * 2.0 ** (old - e)))
                for off, n in members.items():
                    rows[off] = round_e4m3(x[n, h] * 2.0 ** -e)
                out[name + "_exp"][pg, h, nb] = e
    return out


def values(cache):
    """(k, v) [P, Hkv, page, D]: code * scale."""
    got = []
    for n in ("k", "v"):
        block = cache[n].shape[2] // cache[n + "_exp"].shape[2]
        got.append(cache[n] * torch.exp2(cache[n + "_exp"].double()).repeat_interleave(block, 2)[..., None])
    return got


def norm_rotate(x, w, positions, inv_freq, eps):
    """RMSNorm and rotate-half of x [T, H, D] in 64 bits; also |a| + |b| of each rotated pair."""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = x.shape[-1] // 2
    ang = positions.double()[:, None, None] * inv_freq.double()
    a, b = y[..., :half], y[..., half:]
    mag = a.abs() + b.abs()
    return (torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1), torch.cat([mag, mag], -1))


def visible(mode, ctx, Q, vis=None):
    """Per query the visible keys as (A, lo, hi): t < A or lo <= t < hi, all below ctx."""
    if mode == "causal":
        return [(ctx - Q + i + 1, 0, 0) for i in range(Q)]
    if mode == "full":
        return [(ctx, 0, 0)] * Q
    return [(ctx - Q + int(a), ctx - Q + int(lo), ctx - Q + int(hi)) for a, lo, hi in vis]


def attention(q, cache, table, lens, scale, mode="causal", vis=None):
    """(out, weight) [B, Q, Hq, D] float64: the attention over the visible
    keys, and sum p |v| / sum p, what a relative error of the p's or v's acts
    on.  Pages outside the pool hold zero keys and values; other keys take no
    part."""
    B, Q, Hq, D = q.shape
    P, H, page, _ = cache["k"].shape
    kv, vv = values(cache)
    out, wgt = torch.zeros(B, Q, Hq, D, dtype=torch.float64), torch.zeros(B, Q, Hq, D, dtype=torch.float64)
    for b in range(B):
        ctx = min(int(lens[b]), table.shape[1] * page)
        if ctx <= 0:
            continue
        ids = table[b, : -(-ctx // page)].long()
        ok = (ids >= 0) & (ids < P)
        k, v = (torch.where(ok[:, None, None, None], x[ids.clamp(0, P - 1)], torch.zeros((), dtype=torch.float64))
                .transpose(0, 1).reshape(H, -1, D)[:, :ctx] for x in (kv, vv))
        t = torch.arange(ctx)
        for i, (a, lo, hi) in enumerate(visible(mode, ctx, Q, vis)):
            seen = (t < a) | ((t >= lo) & (t < hi))
            if not bool(seen.any()):
                continue
            for h in range(H):
                g = slice(h * (Hq // H), (h + 1) * (Hq // H))
                p = torch.softmax(q[b, i, g].double() @ k[h][seen].t() * scale, -1)
                out[b, i, g] = p @ v[h][seen]
                wgt[b, i, g] = p @ v[h][seen].abs()
    return out, wgt
