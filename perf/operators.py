"""The operators of the 8-bit paged KV cache, and the cases their speed is measured on.

The cache holds keys and values as e4m3 codes with one power-of-two scale for
each block of tokens and KV head (``d3d_amd.fp8_kv``).  Three operators use it:
block attention over it (causal, bidirectional and packed blocks), appending
keys and values to it, and the norm-rotate-append that precedes attention in a
layer.  Head layouts, block sizes and contexts are those of the 8B-shaped
target (32 query heads, 8 KV heads), the 1.7B-shaped draft (16 and 8) and
generic ones; head dimension 128.
"""
import math
import random

import torch

own = False

D = 128
EPS = 1e-6
ROPE_THETA = 1_000_000.0
DEV = "cuda:0"
E_MIN, E_MAX = -117, 119  # exponents of the scales: every stored value is a normal, finite bf16


def listed():
    return [
        # One token of one short conversation: the smallest call, where latency counts.
        dict(name="decode_b1", kind="attn", mode="causal", B=1, Q=1, Hq=32, Hkv=8, lo=333, hi=333, page=16, block=16,
             ctx_seed=1),
        # One request's block of drafted tokens checked by the target.
        dict(name="verify_b1", kind="attn", mode="causal", B=1, Q=16, Hq=32, Hkv=8, lo=2064, hi=2064, page=16,
             block=16, ctx_seed=1),
        # The same for a serving batch of mixed contexts.
        dict(name="verify_b8", kind="attn", mode="causal", B=8, Q=16, Hq=32, Hkv=8, lo=512, hi=8192, page=16,
             block=16, ctx_seed=3),
        # Target-only decoding of a larger batch, a token each.
        dict(name="decode_b48", kind="attn", mode="causal", B=48, Q=1, Hq=32, Hkv=8, lo=256, hi=8191, page=16,
             block=16, ctx_seed=9),
        # The draft's block: it sees its prefix and all of itself.
        dict(name="draft_b4", kind="attn", mode="full", B=4, Q=16, Hq=16, Hkv=8, lo=512, hi=2048, page=16, block=16,
             ctx_seed=4),
        # The draft's packed prediction: a pending block and 16 branches per request.
        dict(name="packed_b4", kind="attn", mode="packed", B=4, Q=272, Hq=16, Hkv=8, lo=512, hi=2048, page=16,
             block=16, ctx_seed=5),
        # Blocks checked far into long documents, large pages, a scale for 64 tokens.
        dict(name="long_b2", kind="attn", mode="causal", B=2, Q=16, Hq=32, Hkv=8, lo=131072, hi=131072, page=256,
             block=64, ctx_seed=2),
        # Prompts as the prefill runs them: slices of 64 tokens, each a request of its own.
        dict(name="prefill_slices", kind="attn", mode="slices", B=2, Q=64, Hq=32, Hkv=8, lo=2500, hi=5500, page=16,
             block=16, ctx_seed=6),
        # A layer's norm, rotation and append for one request's block.
        dict(name="rope_b1", kind="rope", B=1, Q=16, Hq=32, Hkv=8, lo=2051, hi=2051, page=16, block=16, ctx_seed=1),
        # The same for the prompts of four new requests, padded at the front to whole blocks.
        dict(name="rope_prefill", kind="rope", B=4, Q=0, Hq=32, Hkv=8, lo=512, hi=4096, page=16, block=16,
             ctx_seed=11),
        # Keys and values of a batch's blocks, computed elsewhere, appended in the middle of pages.
        dict(name="append_b8", kind="append", B=8, Q=16, Hq=32, Hkv=8, lo=512, hi=4096, page=16, block=16,
             ctx_seed=7),
        # Keys and values of whole prompts (a cache taken over from a bf16 one), larger pages and blocks.
        dict(name="append_prefill", kind="append", B=4, Q=0, Hq=16, Hkv=8, lo=1000, hi=8000, page=64, block=32,
             ctx_seed=8),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "rope", "append"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 8), (16, 8), (8, 8), (16, 2), (12, 4), (40, 8)])
    page = rng.choice([16, 16, 32, 64, 256])
    c = dict(kind=kind, Hq=Hq, Hkv=Hkv, page=page, block=rng.choice([b for b in (16, 32, 64) if b <= page]),
             ctx_seed=rng.randrange(1000))
    if kind == "attn":
        mode = rng.choice(["causal", "causal", "causal", "full", "packed", "slices"])
        if mode == "packed":
            hi, B, Q = _log(rng, 64, 2048), rng.randint(1, 4), 16 * rng.randint(2, 18)
        elif mode == "slices":
            hi, B, Q = _log(rng, 32, 4096), rng.randint(1, 2), rng.choice([16, 64])
        else:
            hi = _log(rng, 32, 65536)
            B, Q = _log(rng, 1, max(1, min(64, 262144 // hi))), rng.choice([1, 1, 16, 16, rng.randint(2, 40)])
        c.update(mode=mode, B=B, Q=Q, lo=max(2, hi // rng.choice([1, 4, 16])), hi=hi)
    else:
        Q = rng.choice([0, 1, 16, rng.randint(2, 40)])
        hi = _log(rng, 32, 4096)
        c.update(B=rng.randint(1, 4) if Q == 0 else _log(rng, 1, 32), Q=Q, lo=max(2, hi // rng.choice([1, 8])), hi=hi)
    return c


# ---------------------------------------------------------------- inputs
def _lens(c):
    r = random.Random(c["ctx_seed"])
    return [_log(r, c["lo"], c["hi"]) for _ in range(c["B"])]


def _vis(c):
    """The packed block's visible keys [Q, 3]: a pending block of 16, then branches of 16 after n of its tokens."""
    r = random.Random(c["ctx_seed"] + 1)
    rows = [(i + 1, 0, 0) for i in range(16)]
    for off in range(16, c["Q"], 16):
        n = r.randint(0, 16)
        rows += [(n, off, off + 16)] * 16
    return rows


def _channels(g, n):
    """Magnitudes of the channels: a few stand out, as the keys' and values' do."""
    m = 0.3 + torch.rand(n, D, generator=g, device=DEV)
    return torch.where(torch.rand(n, D, generator=g, device=DEV) < 0.03, m * 8, m)


def _pow2(byte):
    """The scales 2^(byte - 127)."""
    return byte.to(torch.uint8).view(torch.float8_e8m0fnu).float()


def _need(amax):
    """The least exponent e with amax <= 448 * 2^e, within its bounds."""
    m, ex = torch.frexp(amax)
    return (ex - 9 + (m > 0.875).int()).clamp(E_MIN, E_MAX)


def _codes(x, e):
    y = (x * _pow2(127 - e)).clamp(-448, 448)
    return torch.where(torch.isfinite(x), y, math.nan).to(torch.float8_e4m3fn)


def _cache(g, pages, c):
    """A filled cache: (k, v, k_scale, v_scale)."""
    Hkv, page, blk = c["Hkv"], c["page"], c["block"]
    got = []
    for _ in range(2):
        x = torch.randn(pages, Hkv, page, D, generator=g, device=DEV) * _channels(g, Hkv)[:, None, :]
        x = x.view(pages, Hkv, page // blk, blk, D)
        e = _need(x.abs().amax((-1, -2)))
        got += [_codes(x, e[..., None, None]).view(pages, Hkv, page, D), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)]
    return got[0], got[2], got[1], got[3]


def _tables(g, lens, page):
    """Page tables [B, width] of shuffled pages, and the pool's size."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    at = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    width = max(need)
    start = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEV)[:, None]
    col = torch.arange(width, device=DEV)[None, :]
    table = at[(start + col).clamp(max=pool - 1)]
    return torch.where(col < torch.tensor(need, device=DEV)[:, None], table, 0).contiguous(), pool


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lens(c)
    s = dict(kind=c["kind"], block=c["block"], page=c["page"], Hq=c["Hq"], Hkv=c["Hkv"])
    if c["kind"] == "attn":
        Q = c["Q"]
        if c["mode"] == "slices":
            # Each prompt cut into slices of Q aligned to its end; a slice's context ends with it.
            table, pool = _tables(g, lens, c["page"])
            n = [-(-m // Q) for m in lens]
            table = table.repeat_interleave(torch.tensor(n, device=DEV), 0)
            ctx = [m - Q * (j - 1 - i) for m, j in zip(lens, n) for i in range(j)]
        else:
            ctx = [m + (Q if c["mode"] == "packed" else 0) for m in lens]
            table, pool = _tables(g, ctx, c["page"])
        B = len(ctx)
        s.update(cache=_cache(g, pool, c), table=table.contiguous(), mode=c["mode"],
                 lens=torch.tensor(ctx, dtype=torch.int32, device=DEV), max_ctx=max(ctx),
                 q=torch.randn(B, Q, c["Hq"], D, generator=g, device=DEV).to(torch.bfloat16),
                 vis=torch.tensor(_vis(c), dtype=torch.int32, device=DEV) if c["mode"] == "packed" else None)
        return s
    # New tokens: Q after each prefix, or (Q = 0) whole prompts, padded at the front to whole blocks of 16.
    total = [m + c["Q"] for m in lens]
    table, pool = _tables(g, total, c["page"])
    pos, row = [], []
    for b, m in enumerate(lens):
        p = torch.arange(m, m + c["Q"]) if c["Q"] else torch.arange(m - -(-m // 16) * 16, m)
        pos.append(p)
        row.append(torch.full_like(p, b))
    pos, row = torch.cat(pos).to(DEV), torch.cat(row).to(DEV)
    at = pos.clamp(min=0)
    slots = table.long()[row, at // c["page"]] * c["page"] + at % c["page"]
    slots = torch.where(pos >= 0, slots, -1).contiguous()
    T, Hq, Hkv = pos.numel(), c["Hq"], c["Hkv"]
    s.update(cache=_cache(g, pool, c), slots=slots, pos=pos.contiguous())
    if c["kind"] == "rope":
        x = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=DEV) * _channels(g, Hq + 2 * Hkv)
        s["qkv"] = x.to(torch.bfloat16).view(T, -1)
        s["qn"], s["kn"] = ((1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2))
        s["inv_freq"] = 1.0 / ROPE_THETA ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float32) / D)
    else:
        s["k"], s["v"] = ((torch.randn(T, Hkv, D, generator=g, device=DEV) * _channels(g, Hkv)).to(torch.bfloat16)
                          for _ in range(2))
    return s


# ---------------------------------------------------------------- the operators
def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "attn":
        return _attend(s)
    if s["kind"] == "rope":
        q, k, v = _rope(s)
    else:
        q, k, v = None, s["k"].float(), s["v"].float()
    _append(s, s["cache"][0], s["cache"][2], k)
    _append(s, s["cache"][1], s["cache"][3], v)
    return [*s["cache"], q] if q is not None else list(s["cache"])


def _run_own(s):
    from d3d_amd import fp8_kv
    if "kv" not in s:
        s["kv"] = fp8_kv.Fp8KV(*s["cache"])  # the cache object that a program keeps
    kv = s["kv"]
    if s["kind"] == "rope":
        q = fp8_kv.qk_rope_append(s["qkv"], s["pos"], s["qn"], s["kn"], s["inv_freq"], kv, s["slots"], s["Hq"],
                                  s["Hkv"], EPS)
        return [kv.k, kv.v, kv.k_scale, kv.v_scale, q]
    if s["kind"] == "append":
        fp8_kv.kv_append(s["k"], s["v"], kv, s["slots"])
        return [kv.k, kv.v, kv.k_scale, kv.v_scale]
    if s["mode"] == "packed":
        return fp8_kv.packed_block_attn(s["q"], kv, s["lens"], s["table"], s["vis"], max_seqlen_k=s["max_ctx"])
    return fp8_kv.flash_attn_with_kvcache(s["q"], kv, s["lens"], s["table"], causal=s["mode"] != "full",
                                          max_seqlen_k=s["max_ctx"])


def _attend(s):
    k8, v8, ks, vs = s["cache"]
    q, table, blk = s["q"], s["table"].long(), s["block"]
    B, Q, Hq, _ = q.shape
    Hkv, S = s["Hkv"], table.shape[1] * s["page"]
    G = Hq // Hkv

    def read(code, scale):  # [B, Hkv, S, D] fp32
        x = code.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x = x.view(B, -1, Hkv, s["page"] // blk, blk, D) * _pow2(scale.view(torch.uint8)[table])[..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, S, D)

    t = torch.arange(S, device=DEV)
    n = s["lens"].long()[:, None, None]
    i = torch.arange(Q, device=DEV)[None, :, None]
    if s["mode"] == "full":
        seen = (t < n).expand(B, Q, S)
    elif s["mode"] == "packed":
        a, lo, hi = (s["vis"].long()[None, :, j, None] + n - Q for j in range(3))
        seen = ((t < a) | ((t >= lo) & (t < hi))) & (t < n)
    else:
        seen = t <= n - Q + i
    seen = seen[:, None, None].expand(B, Hkv, G, Q, S).reshape(B, Hkv, G * Q, S)
    qh = q.float().view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    score = torch.matmul(qh, read(k8, ks).transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, read(v8, vs)) / torch.where(total == 0, 1.0, total)
    return out.view(B, Hkv, G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D).to(torch.bfloat16)


def _rope(s):
    Hq, Hkv = s["Hq"], s["Hkv"]
    x = s["qkv"].float().view(-1, Hq + 2 * Hkv, D)
    turn = s["pos"].double()[:, None] * s["inv_freq"].double()  # far positions: the angle in 64 bits
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]

    def rotate(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y[..., : D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    return rotate(x[:, :Hq], s["qn"]).to(torch.bfloat16), rotate(x[:, Hq:Hq + Hkv], s["kn"]), x[:, Hq + Hkv:]


def _append(s, code, scale, x):
    """x [T, Hkv, D] fp32 into the blocks that its slots touch."""
    blk, page = s["block"], s["page"]
    live = (s["slots"] >= 0).nonzero()[:, 0]
    slots, x = s["slots"][live], x[live]
    at, which = torch.unique(slots // blk, return_inverse=True)
    pg, nb = at // (page // blk), at % (page // blk)
    n, Hkv = at.numel(), x.shape[1]
    raw = code.view(torch.uint8).view(code.shape[0], Hkv, page // blk, blk, D)
    exps = scale.view(torch.uint8)
    amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    top = torch.zeros(n, Hkv, device=DEV).index_reduce_(0, which, amax, "amax")
    need = _need(top) + 127
    old = exps[pg, :, nb].int()
    first = torch.zeros(n, dtype=torch.bool, device=DEV).index_fill_(0, which[slots % blk == 0], True)
    new = torch.where(first[:, None], need, torch.maximum(old, need))
    kept = raw[pg, :, nb].view(torch.float8_e4m3fn).float() * _pow2((old - new + 127).clamp(0, 254))[..., None, None]
    kept = torch.where(first[:, None, None, None], 0.0, kept).to(torch.float8_e4m3fn).view(torch.uint8)
    kept[which, :, slots % blk] = _codes(x, new[which][..., None] - 127).view(torch.uint8)
    raw[pg, :, nb] = kept
    exps[pg, :, nb] = new.to(torch.uint8)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, lens = case, _lens(case)
    Hq, Hkv, Q = c["Hq"], c["Hkv"], c["Q"]
    if c["kind"] == "attn":
        if c["mode"] == "slices":
            rows = sum(-(-n // Q) * Q for n in lens)
            keys, pairs, tabs = sum(lens), sum(n * (n + 1) // 2 for n in lens), sum(-(-n // Q) * -(-n // c["page"]) for n in lens)
        else:
            ctx = [n + (Q if c["mode"] == "packed" else 0) for n in lens]
            rows, keys, tabs = Q * c["B"], sum(ctx), sum(-(-n // c["page"]) for n in ctx)
            if c["mode"] == "causal":
                pairs = sum(max(0, n - Q + i + 1) for n in ctx for i in range(Q))
            elif c["mode"] == "full":
                pairs = Q * sum(ctx)
            else:
                pairs = sum(n + a + hi - lo for n in lens for a, lo, hi in _vis(c))
        moved = keys * Hkv * 2 * (D + 1 / c["block"]) + 2 * rows * Hq * D * 2 + 4 * tabs + 4 * c["B"]
        return {"bytes": moved, "flops": 4.0 * D * Hq * pairs}
    T = sum(lens) if Q == 0 else Q * c["B"]
    rows = sum(-(-n // 16) * 16 for n in lens) if Q == 0 else T
    moved = T * Hkv * 2 * D + 8 * rows
    if c["kind"] == "rope":
        return {"bytes": moved + rows * (Hq + 2 * Hkv) * D * 2 + rows * Hq * D * 2 + 8 * rows,
                "flops": 8.0 * rows * (Hq + Hkv) * D}
    return {"bytes": moved + T * Hkv * 2 * D * 2, "flops": 3.0 * T * Hkv * 2 * D}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attn(s) if s["kind"] == "attn" else _exact_append(s)


def _exact_attn(s):
    q = s["q"].double()
    B, Q, Hq, _ = q.shape
    G, page = Hq // s["Hkv"], s["page"]
    out = torch.zeros_like(q)
    vis = s["vis"].tolist() if s["vis"] is not None else None
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : -(-n // page)].long()
        if vis is not None:
            row = [(n - Q + a, n - Q + lo, n - Q + hi) for a, lo, hi in vis]
        else:
            row = [(n if s["mode"] == "full" else n - Q + i + 1, 0, 0) for i in range(Q)]
        lim = torch.tensor(row, device=DEV)
        t = torch.arange(n, device=DEV)
        hide = ~((t < lim[:, :1]) | ((t >= lim[:, 1:2]) & (t < lim[:, 2:])))
        for h in range(s["Hkv"]):
            kv = []
            for code, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1], s["cache"][3])):
                x = code[:, h].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
                e = scale[:, h].contiguous().view(torch.uint8)[pages].double() - 127
                kv.append((x * torch.exp2(e).repeat_interleave(s["block"], 1)[..., None]).reshape(-1, D)[:n])
            for j in range(h * G, (h + 1) * G):
                z = (q[b, :, j] @ kv[0].t()) / math.sqrt(D)
                z = z.masked_fill(hide, -math.inf)
                out[b, :, j] = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) @ kv[1]
    return out


def _round8(y):
    """y rounded to the nearest e4m3 value, ties to even, in 64 bits."""
    a = y.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.where(torch.isfinite(y), torch.sign(y) * torch.round(a / step) * step, math.nan)


def _exact_append(s):
    blk, page, Hq, Hkv = s["block"], s["page"], s["Hq"], s["Hkv"]
    q = None
    if s["kind"] == "rope":
        x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
        ang = s["pos"].double()[:, None, None] * s["inv_freq"].double()

        def turned(x, w):
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(y[..., : D // 2], y[..., D // 2:]) * torch.polar(torch.ones_like(ang), ang)
            return torch.cat([z.real, z.imag], -1)

        q, k, v = turned(x[:, :Hq], s["qn"]), turned(x[:, Hq:Hq + Hkv], s["kn"]), x[:, Hq + Hkv:]
    else:
        k, v = s["k"].double(), s["v"].double()
    live = s["slots"] >= 0
    slots = s["slots"][live]
    pg, off = slots // page, slots % page
    codes, scales = [], []
    for x, code, scale in ((k[live], s["cache"][0], s["cache"][2]), (v[live], s["cache"][1], s["cache"][3])):
        P = code.shape[0]
        # Over the whole pool: the largest new entry of each block, and which blocks start anew.
        new = torch.zeros(P, Hkv, page, D, dtype=torch.float64, device=DEV)
        wrote = torch.zeros(P, page, dtype=torch.bool, device=DEV)
        new[pg, :, off] = x
        wrote[pg, off] = True
        most = new.abs().view(P, Hkv, page // blk, -1).amax(-1)
        e = torch.ceil(torch.log2(most / 448)).clamp(E_MIN, E_MAX)
        e = torch.where(most > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(most <= 448 * torch.exp2(e - 1), e - 1, e).clamp(E_MIN, E_MAX)
        touched = wrote.view(P, 1, page // blk, blk).any(-1)
        anew = wrote.view(P, 1, page // blk, blk)[..., 0]
        had = scale.view(torch.uint8).double() - 127
        e = torch.where(anew, e, torch.where(touched, torch.maximum(had, e), had))
        was = torch.where(anew[..., None, None], 0.0, code.double().view(P, Hkv, page // blk, blk, D)) * torch.exp2(had - e)[..., None, None]
        now = torch.where(wrote.view(P, 1, page // blk, blk, 1), new.view(P, Hkv, page // blk, blk, D) * torch.exp2(-e)[..., None, None], was)
        codes.append(_round8(now).view(P, Hkv, page, D))
        scales.append(torch.exp2(e))
    return [*codes, *scales, q] if q is not None else [*codes, *scales]
