"""The 8-bit paged cache against its 64-bit oracle (GPU).

* Appends of bf16 rows have one right answer, bit for bit: amax, the exponent
  and the rounding are exact in fp32.
* After norm and rotation a value x is known to 2^-17 (|a| + |b|) of its rotated
  pair (fp32 sums, rsqrt, sine and cosine); a query adds half a bf16 step, 2^-8 |x|, a key half an e4m3 step,
  2^-4 |x|, or 2^-10 of its scale below the normal range.
* An attention output is off by half a bf16 step, 2^-8 |o|, and by the
  rounding of the probabilities to bf16 (each at most 2^-8 of itself) and fp32
  scores and sums (2^-10 together) acting on sum p |v| / sum p.
"""
from __future__ import annotations

import math

import pytest
import torch

from d3d_amd import _lib, fp8_kv
from d3d_amd import attention as att
from d3d_amd import layers as ly
from d3d_amd.fp8_kv import Fp8KV
from oracle import fp8_kv as of

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BF = torch.bfloat16
D = 128


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _filled(g, P, H, page, block, spread=3.0):
    """A cache of random codes and scales (no NaN)."""
    n = P * H * page * D
    codes = [torch.randint(0, 256, (n,), generator=g, dtype=torch.int64) for _ in range(2)]
    codes = [torch.where(c % 128 == 127, c - 1, c).to(torch.uint8).view(torch.float8_e4m3fn).view(P, H, page, D)
             for c in codes]
    scales = [(127 - 7 + spread * torch.randn(P, H, page // block, generator=g)).round().to(torch.uint8)
              .view(torch.float8_e8m0fnu) for _ in range(2)]
    return codes + scales


def _like_data(g, P, H, page, block):
    """A cache quantised from normal entries, as appends leave it."""
    got = []
    for _ in range(2):
        x = torch.randn(P, H, page // block, block, D, generator=g) * torch.rand(H, 1, 1, D, generator=g)
        amax = x.abs().amax((-1, -2))
        m, ex = torch.frexp(amax)
        e = ex - 9 + (m > 0.875).int()
        got.append(((x * torch.exp2(-e[..., None, None].float())).to(torch.float8_e4m3fn).view(P, H, page, D),
                    (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)))
    return [got[0][0], got[1][0], got[0][1], got[1][1]]


def _to_dev(parts):
    return Fp8KV(*(t.view(torch.uint8).to(DEV).view(t.dtype) for t in parts))


def _same_cache(cache, want):
    for n, code, scale in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
        exps = scale.cpu().view(torch.uint8).long() - 127
        assert torch.equal(exps, want[n + "_exp"]), n
        got, ref = code.cpu().double(), want[n]
        assert torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), ref.nan_to_num(nan=0.0)), n


# ------------------------------------------------------------------ appends
@pytest.mark.parametrize("P,H,page,block", [(6, 2, 16, 16), (5, 8, 64, 16), (4, 1, 64, 32), (3, 3, 64, 64),
                                            (3, 2, 256, 128), (2, 2, 256, 256), (5, 2, 48, 16), (3, 1, 96, 32)])
@pytest.mark.parametrize("order", ["run", "shuffled", "repeated"])
def test_kv_append(P, H, page, block, order):
    g = _gen(P * 1000 + page + block)
    parts = _filled(g, P, H, page, block)
    total = P * page
    if order == "run":  # ends inside a block, starts inside one, with slots to skip
        slots = torch.arange(page // 2 + 3, min(total, page // 2 + 3 + 70))
        slots[::13] = -1
    elif order == "shuffled":
        slots = torch.randperm(total, generator=g)[: total // 3]
        slots = torch.cat([slots, torch.tensor([-5, total, total + 7, 2 ** 40, -2 ** 40])])
        slots = slots[torch.randperm(len(slots), generator=g)]
    else:  # every slot several times, the last one counts
        slots = torch.randint(0, total // 2, (total,), generator=g)
    N = len(slots)
    k = (torch.randn(N, H, D, generator=g) * torch.exp2(torch.randint(-12, 6, (N, 1, 1), generator=g).float())).to(BF)
    v = torch.randn(N, H, D, generator=g).to(BF)
    cache = _to_dev(parts)
    fp8_kv.kv_append(k.to(DEV), v.to(DEV), cache, slots.to(DEV))
    _same_cache(cache, of.append(of.from_bytes(*parts), k.double(), v.double(), slots))


def test_kv_append_many_tokens_across_windows():
    """Over 1,024 tokens a workgroup leads several blocks: whole prompts in
    order, with padding in front, and the same slots scattered."""
    g = _gen(5)
    parts = _filled(g, 110, 2, 16, 16)
    slots = torch.cat([torch.full((9,), -1), torch.arange(5, 1500)])
    for s in (slots, slots[torch.randperm(len(slots), generator=g)]):
        k, v = (torch.randn(len(s), 2, D, generator=g).to(BF) for _ in range(2))
        cache = _to_dev(parts)
        fp8_kv.kv_append(k.to(DEV), v.to(DEV), cache, s.to(DEV))
        _same_cache(cache, of.append(of.from_bytes(*parts), k.double(), v.double(), s))


@pytest.mark.parametrize("T,Hkv,page,block", [(300, 1, 16, 16), (1500, 1, 16, 16), (5000, 1, 64, 16), (9000, 1, 64, 32),
                                              (700, 2, 64, 64), (2500, 1, 256, 256), (17000, 1, 128, 128)])
def test_kv_append_of_scattered_calls(T, Hkv, page, block):
    """Calls of every length class, their tokens in any order over blocks filled
    before, some outside the cache and some slots twice."""
    g = _gen(T)
    P = T // page + 3
    parts = _filled(g, P, Hkv, page, block)
    slots = torch.randperm(P * page, generator=g)[:T]
    slots[torch.randint(0, T, (T // 20,), generator=g)] = slots[0].clone()
    slots[torch.randint(0, T, (T // 50,), generator=g)] = -1
    slots[torch.randint(0, T, (T // 50,), generator=g)] = P * page
    k, v = (torch.randn(T, Hkv, D, generator=g).to(BF) for _ in range(2))
    cache = _to_dev(parts)
    fp8_kv.kv_append(k.to(DEV), v.to(DEV), cache, slots.to(DEV))
    want = of.append(of.from_bytes(*parts), k.double(), v.double(), slots)
    got = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for n in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("block", [16, 64])
def test_kv_append_token_by_token(block):
    """Growing, rewinding and starting a block anew, one call at a time."""
    g = _gen(block)
    cache, want = Fp8KV.empty(2, 64, 2, DEV, block=block), of.empty(2, 2, 64, block)
    for step, n in enumerate([0, 1, 2, 3, 2, 3, 4, 15, 16, 17, 18, 16, 0, 1, 63, 64, 70]):
        k = (torch.randn(1, 2, D, generator=g) * 2.0 ** (step % 7 * 3 - 9)).to(BF)
        v = (torch.randn(1, 2, D, generator=g) * 2.0 ** (9 - step % 5 * 4)).to(BF)
        fp8_kv.kv_append(k.to(DEV), v.to(DEV), cache, torch.tensor([n], device=DEV))
        want = of.append(want, k.double(), v.double(), [n])
        _same_cache(cache, want)


def test_kv_append_extremes():
    """Zeros, NaN, infinities, the smallest and the largest bf16, and ties."""
    k = torch.zeros(8, 1, D)
    k[1] = torch.arange(D).float() * 2.0 ** -133      # denormal bf16
    k[2, 0, ::3] = math.inf
    k[3, 0, 1] = math.nan
    k[3, 0, 5] = -3.3e38
    k[4] = 3.38e38
    k[5] = 448.0
    k[6] = 449.0 * torch.where(torch.arange(D) % 2 == 0, 1.0, -1.0)
    k[7] = 1.0 + torch.arange(D).float() / 128        # ties of e4m3 among them
    k = k.to(BF)
    for rows in ([0], [1], [2], [3], [4], [5], [6], [7], [0, 1, 7], list(range(8))):
        cache, want = Fp8KV.empty(2, 16, 1, DEV), of.empty(2, 1, 16, 16)
        for first in (16, 17):  # anew, then kept entries that may have to move
            slots = torch.arange(first, first + len(rows))
            x = k[rows]
            fp8_kv.kv_append(x.to(DEV), x.flip(-1).to(DEV), cache, slots.to(DEV))
            want = of.append(want, x.double(), x.flip(-1).double(), slots)
            _same_cache(cache, want)
        for t in cache.dequantize():  # every stored value is a finite bf16 or NaN
            assert not t.isinf().any()


def test_kv_append_strided_rows_and_other_types():
    """Slices of a fused qkv product, flat rows, int32 slots, no tokens."""
    g = _gen(8)
    parts = _filled(g, 4, 2, 16, 16)
    qkv = torch.randn(20, 8, D, generator=g).to(BF)
    slots = torch.arange(7, 27)
    want = of.append(of.from_bytes(*parts), qkv[:, 4:6].double(), qkv[:, 6:].double(), slots)
    d = qkv.to(DEV)
    for k, v in ((d[:, 4:6], d[:, 6:]), (d.view(20, -1)[:, 512:768], d.view(20, -1)[:, 768:]),
                 (d[:, 4:6].transpose(0, 1).contiguous().transpose(0, 1), d[:, 6:].contiguous()),
                 (d[:, 4:6].float(), d[:, 6:])):
        cache = _to_dev(parts)
        fp8_kv.kv_append(k, v, cache, slots.to(DEV, torch.int32))
        _same_cache(cache, want)
    fp8_kv.kv_append(d[:0, 4:6], d[:0, 6:], cache, slots[:0].to(DEV))
    _same_cache(cache, want)
    with pytest.raises(ValueError, match="tokens"):
        fp8_kv.kv_append(d[:, 4:7], d[:, 6:], cache, slots.to(DEV))


def test_append_and_attend_past_32_bit_offsets():
    """Pages whose bytes lie past 2^32."""
    P, H, page = (1 << 32) // (8 * 64 * D) + 40, 8, 64
    cache = Fp8KV.empty(P, page, H, DEV, block=16)
    g = _gen(4)
    pages = [P - 1, P - 37, 3]
    slots = torch.cat([torch.arange(p * page, (p + 1) * page) for p in pages])[:150]
    k, v = (torch.randn(150, H, D, generator=g).to(BF) for _ in range(2))
    fp8_kv.kv_append(k.to(DEV), v.to(DEV), cache, slots.to(DEV))
    pick = torch.tensor(pages, device=DEV)
    small = [t.view(torch.uint8)[pick].cpu().view(t.dtype) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    want = of.append(of.empty(3, H, page, 16), k.double(), v.double(), torch.arange(150))
    _same_cache(_to_dev(small), want)
    assert int(cache.k.view(torch.uint8).view(torch.int32).count_nonzero()) <= 150 * H * D // 4
    q = torch.randn(1, 5, 16, D, generator=g).to(BF)
    out = fp8_kv.flash_attn_with_kvcache(q.to(DEV), cache, torch.tensor([150], device=DEV), pick[None].int())
    _close(out, *of.attention(q, want, torch.arange(3)[None], [150], D ** -0.5))


# ---------------------------------------------------- norm, rotation and append
def _rope_inputs(g, T, Hq, Hkv):
    qkv = (torch.randn(T, Hq + 2 * Hkv, D, generator=g) * 2).to(BF)
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g)).to(BF) for _ in range(2))
    inv_freq = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
    return qkv, qn, kn, inv_freq


def _check_rope(q, cache, before, qkv, pos, qn, kn, inv_freq, slots, Hq, Hkv, eps):
    """slots distinct and every touched block started anew or filled before."""
    x = qkv.double()
    rq, mag = of.norm_rotate(x[:, :Hq], qn, pos, inv_freq, eps)
    err = (q.cpu().double() - rq).abs()
    assert bool((err <= 2.0 ** -8 * rq.abs() + 2.0 ** -17 * mag).all()), float((err - 2.0 ** -8 * rq.abs()).max())
    rk, kmag = of.norm_rotate(x[:, Hq:Hq + Hkv], kn, pos, inv_freq, eps)
    want = of.append(before, rk, x[:, Hq + Hkv:], slots)
    assert torch.equal(cache.v.cpu().double(), want["v"])
    assert torch.equal(cache.v_scale.cpu().view(torch.uint8).long() - 127, want["v_exp"])
    # A key's exponent may differ only where its block's amax is within fp32's reach of a border.
    got = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
    page, block = got["k"].shape[2], cache.block
    off = (got["k_exp"] != want["k_exp"]).nonzero().tolist()
    top = {}
    for n, s in enumerate(slots.tolist()):
        if 0 <= s:
            for h in range(Hkv):
                at = (s // page, h, s % page // block)
                top[at] = max(top.get(at, 0.0), float(rk[n, h].abs().max()))
    for at in off:
        a = top[tuple(at)]
        assert of.need_exp(a * (1 - 2.0 ** -14)) != of.need_exp(a * (1 + 2.0 ** -14)), at
    kv = of.values(got)[0]
    scale = torch.exp2(got["k_exp"].double()).repeat_interleave(block, 2)[..., None]
    live = slots >= 0
    pg, sl = slots[live] // page, slots[live] % page
    err = (kv[pg, :, sl] - rk[live]).abs()
    tol = torch.maximum(2.0 ** -4 * rk[live].abs(), 2.0 ** -10 * scale.expand_as(kv)[pg, :, sl]) + 2.0 ** -16 * kmag[live]
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("T,Hq,Hkv,page,block,first", [
    (1, 32, 8, 16, 16, 2051), (16, 32, 8, 16, 16, 0), (16, 16, 8, 16, 16, 2051), (37, 16, 2, 64, 64, 5),
    (5, 3, 3, 32, 32, 31), (200, 12, 4, 256, 128, 130), (300, 8, 8, 256, 256, 7), (1100, 20, 4, 16, 16, 3),
])
def test_qk_rope_append(T, Hq, Hkv, page, block, first):
    g = _gen(T + Hq)
    qkv, qn, kn, inv_freq = _rope_inputs(g, T, Hq, Hkv)
    P = (first + T) // page + 2
    parts = _filled(g, P, Hkv, page, block, spread=0.0)
    perm = torch.randperm(P, generator=g)
    pos = torch.arange(first, first + T)
    slots = perm[pos // page] * page + pos % page
    if T > 20:
        slots[:3] = -1  # padding rows: no place in the cache, a query all the same
    cache = _to_dev(parts)
    q = fp8_kv.qk_rope_append(qkv.view(T, -1).to(DEV), pos.to(DEV), qn.to(DEV), kn.to(DEV), inv_freq.to(DEV), cache,
                              slots.to(DEV), Hq, Hkv, 1e-6)
    _check_rope(q, cache, of.from_bytes(*parts), qkv, pos, qn, kn, inv_freq, slots, Hq, Hkv, 1e-6)


def test_qk_rope_append_far_positions():
    """Angles of positions past 2^24, which a float cannot hold, and negative ones."""
    T, Hq, Hkv = 16, 4, 2
    g = _gen(9)
    qkv, qn, kn, inv_freq = _rope_inputs(g, T, Hq, Hkv)
    pos = torch.tensor([0, 1, -1, -15, 131071, 1_000_003, 2 ** 24 + 1, 2 ** 24 + 3, 2 ** 26 + 5, 10 ** 8 + 7, 2 ** 28 - 1,
                        5, 6, 7, 8, 9])
    slots = torch.arange(16)
    parts = _filled(g, 1, Hkv, 16, 16)
    cache = _to_dev(parts)
    q = fp8_kv.qk_rope_append(qkv.view(T, -1).to(DEV), pos.to(DEV), qn.to(DEV), kn.to(DEV), inv_freq.to(DEV), cache,
                              slots.to(DEV), Hq, Hkv, 1e-5)
    _check_rope(q, cache, of.from_bytes(*parts), qkv, pos, qn, kn, inv_freq, slots, Hq, Hkv, 1e-5)


@pytest.mark.parametrize("T,splits", [(1, 2), (16, 4), (64, 7)])
def test_qk_rope_append_of_split_products(T, splits):
    """Split partials give what their rounded sum gives, bit for bit."""
    Hq, Hkv = 8, 2
    g = _gen(T)
    _, qn, kn, inv_freq = _rope_inputs(g, 1, Hq, Hkv)
    parts = torch.randn(splits, T, (Hq + 2 * Hkv) * D, generator=g).to(DEV)
    prod = ly.SplitProduct(parts, splits)
    pos, slots = torch.arange(11, 11 + T, device=DEV), torch.arange(3, 3 + T, device=DEV)
    filled = _filled(g, 6, Hkv, 16, 16)
    a, b = _to_dev(filled), _to_dev(filled)
    args = (pos, qn.to(DEV), kn.to(DEV), inv_freq.to(DEV))
    qa = fp8_kv.qk_rope_append(prod, *args, a, slots, Hq, Hkv, 1e-6)
    qb = fp8_kv.qk_rope_append(prod.value(), *args, b, slots, Hq, Hkv, 1e-6)
    assert torch.equal(qa, qb)
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("T,page,block,first", [(48, 16, 16, 0), (600, 16, 16, 4096), (600, 64, 64, 65536), (130, 256, 256, 256)])
def test_rotated_keys_are_the_exact_ones(T, page, block, first):
    """Normalised, rotated and scaled in 64 bits and rounded once, keys get the
    codes of the formula: 2^-35 of a value, what 64-bit angles of these positions
    leave, meets one of its 16 borders per octave at fewer than 1 in 10^8 values."""
    g = _gen(T + page)
    Hq, Hkv = 8, 8
    qkv, qn, kn, inv_freq = _rope_inputs(g, T, Hq, Hkv)
    pos = torch.arange(first, first + T)
    P = -(-T // page)
    slots = torch.randperm(P, generator=g)[torch.arange(T) // page] * page + torch.arange(T) % page
    cache = Fp8KV.empty(P, page, Hkv, DEV, block=block)
    before = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
    fp8_kv.qk_rope_append(*(t.to(DEV) for t in (qkv.view(T, -1), pos, qn, kn, inv_freq)), cache, slots.to(DEV), Hq, Hkv, 1e-6)
    x = qkv.double()
    rk, _ = of.norm_rotate(x[:, Hq:Hq + Hkv], kn, pos, inv_freq, 1e-6)
    want = of.append(before, rk, x[:, Hq + Hkv:], slots)
    got = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for n in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(got[n], want[n]), n


def test_qk_rope_append_refusals():
    g = _gen(1)
    qkv, qn, kn, inv_freq = (t.to(DEV) for t in _rope_inputs(g, 4, 4, 2))
    cache = Fp8KV.empty(2, 16, 2, DEV)
    at = torch.arange(4, device=DEV)
    good = dict(qkv=qkv.view(4, -1), positions=at, q_norm=qn, k_norm=kn, inv_freq=inv_freq, cache=cache, slot_mapping=at,
                heads=4, kv_heads=2, eps=1e-6)
    fp8_kv.qk_rope_append(**good)
    for bad in (dict(qkv=qkv.view(4, -1).float()), dict(qkv=qkv.view(4, -1)[:, :-D]), dict(kv_heads=1), dict(heads=3),
                dict(positions=at.int()), dict(slot_mapping=at[:3]), dict(q_norm=qn[:64]), dict(k_norm=kn.float()),
                dict(inv_freq=inv_freq.double()), dict(inv_freq=inv_freq[:32]),
                dict(q_out=torch.empty(4, 4, D, device=DEV)), dict(qkv=qkv.view(4, -1).t().contiguous().t())):
        with pytest.raises(ValueError):
            fp8_kv.qk_rope_append(**{**good, **bad})


@pytest.mark.parametrize("n", (1, 3))
def test_append_of_rows_at_odd_strides_and_addresses(n):
    """Rows whose stride or address the kernel does not take, also of a single
    token, whose stride no layout test looks at."""
    g = _gen(61)
    wide = torch.randn(8 * 1027, generator=g).to(BF)
    slots = torch.tensor([5, 21, 40])[:n]
    for at, step in ((0, 1027), (1, 1024), (2, 1026), (4, 1024), (3, 1025)):
        rows = torch.as_strided(wide, (n, 8, D), (step, D, 1), at)
        dev = torch.as_strided(wide.to(DEV), (n, 8, D), (step, D, 1), at)
        got, want = (Fp8KV.empty(3, 16, 8, DEV) for _ in range(2))
        fp8_kv.kv_append(dev, dev, got, slots.to(DEV))
        fp8_kv.kv_append(rows.clone(memory_format=torch.contiguous_format).to(DEV), rows.to(DEV).clone(
            memory_format=torch.contiguous_format), want, slots.to(DEV))
        assert got.k.view(torch.uint8).any()
        for a, b in ((got.k, want.k), (got.v, want.v), (got.k_scale, want.k_scale), (got.v_scale, want.v_scale)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ------------------------------------------------------------------ attention
def _close(out, ref, wgt):
    got = out.cpu().double()
    assert torch.equal(got.isnan(), ref.isnan()), "NaN in other places"
    ref, wgt = ref.nan_to_num(nan=0.0), wgt.nan_to_num(nan=0.0)
    err = (got.nan_to_num(nan=0.0) - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * wgt
    assert bool((err <= tol).all()), f"off by {float((err / tol.clamp(min=1e-30)).max()):.2f} of the tolerance"


def _attend(q, cache, lens, table, mode, vis=None, **kw):
    lens, table = torch.as_tensor(lens), table
    if mode == "packed":
        return fp8_kv.packed_block_attn(q.to(DEV), cache, lens.to(DEV), table.to(DEV),
                                        torch.tensor(vis, dtype=torch.int32, device=DEV), **kw)
    return fp8_kv.flash_attn_with_kvcache(q.to(DEV), cache, lens.to(DEV), table.to(DEV), causal=mode == "causal", **kw)


def _case(seed, lens, Q, Hq, Hkv, page, block, mode, vis=None, sharp=1.0, **kw):
    g = _gen(seed)
    width = max(1, max(-(-n // page) for n in lens))
    need = sum(-(-max(n, 0) // page) for n in lens)
    P = need + 2
    parts = _like_data(g, P, Hkv, page, block)
    perm = torch.randperm(P, generator=g)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        for j in range(-(-max(n, 0) // page)):
            table[b, j] = perm[at]
            at += 1
    q = (torch.randn(len(lens), Q, Hq, D, generator=g) * sharp).to(BF)
    out = _attend(q, _to_dev(parts), lens, table, mode, vis, **kw)
    _close(out, *of.attention(q, of.from_bytes(*parts), table, lens, D ** -0.5, mode, vis))


@pytest.mark.parametrize("lens,Q,Hq,Hkv,page,block", [
    ([1], 1, 8, 8, 16, 16), ([1], 1, 32, 8, 16, 16), ([17], 1, 32, 8, 16, 16), ([333], 1, 32, 8, 16, 16),
    ([31, 32, 33, 64, 65, 127, 128, 129], 1, 16, 8, 16, 16),
    ([2064], 16, 32, 8, 16, 16), ([3000], 16, 16, 8, 64, 32), ([700, 40, 1, 0, 1999], 16, 32, 8, 16, 16),
    ([100, 7], 3, 12, 4, 48, 16), ([513, 255], 2, 64, 1, 32, 32), ([400], 5, 40, 8, 256, 256),
    ([129, 300], 9, 8, 8, 128, 128), ([257], 64, 32, 8, 16, 16), ([90], 100, 8, 2, 16, 16), ([600], 33, 16, 2, 64, 64),
    ([5000], 1, 8, 1, 256, 64), ([9000, 12], 16, 16, 2, 16, 16),
])
@pytest.mark.parametrize("mode", ["causal", "full"])
def test_attention(lens, Q, Hq, Hkv, page, block, mode):
    _case(len(lens) * 100 + Q, lens, Q, Hq, Hkv, page, block, mode)


@pytest.mark.parametrize("lens", [[5] * 70, [(37 * i) % 900 for i in range(80)]])
def test_attention_of_many_requests(lens):
    _case(7, lens, 1, 8, 2, 16, 16, "causal")


@pytest.mark.parametrize("sharp", [0.0, 8.0, 60.0])
def test_attention_flat_and_peaked(sharp):
    """Equal scores, and scores whose largest outweighs everything."""
    _case(11, [1500, 77], 4, 8, 2, 16, 16, "causal", sharp=sharp)


@pytest.mark.parametrize("Hq,Hkv,Q,n", [(8, 8, 1, 333), (16, 2, 1, 500), (32, 8, 2, 90), (16, 8, 8, 257)])
def test_attention_of_few_rows_keeps_the_results_rounding(Hq, Hkv, Q, n):
    """Up to 16 rows of a KV head over one range: probabilities are held to 2^-17
    and fp32 scores (log2, below 2^8) to 2^-15, so that beside the result's half
    step there is 2^-13 of the values at most, peaked rows included."""
    g = _gen(n)
    P = -(-n // 16) + 1
    parts = _like_data(g, P, Hkv, 16, 16)
    table = torch.randperm(P, generator=g)[None, :P].int()
    for sharp in (1.0, 4.0, 12.0):
        q = (torch.randn(1, Q, Hq, D, generator=g) * sharp).to(BF)
        got = _attend(q, _to_dev(parts), [n], table, "causal").cpu().double()
        ref, wgt = of.attention(q, of.from_bytes(*parts), table, [n], D ** -0.5)
        assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -13 * wgt).all())


def test_attention_late_maximum():
    """The largest score at the very end and at the very start of a long context."""
    g = _gen(3)
    parts = _like_data(g, 260, 1, 16, 16)
    for at in (0, 4095, 2048):
        k = parts[0].clone().view(torch.uint8)
        k[at // 16, 0, at % 16] = torch.tensor([448.0]).to(torch.float8_e4m3fn).view(torch.uint8)
        p = [k.view(torch.float8_e4m3fn), *parts[1:]]
        q = torch.ones(1, 2, 4, D).to(BF)
        table = torch.arange(260, dtype=torch.int32)[None]
        out = _attend(q, _to_dev(p), [4096], table, "full")
        _close(out, *of.attention(q, of.from_bytes(*p), table, [4096], D ** -0.5, "full"))


@pytest.mark.parametrize("lens,K,accepted,Hq,Hkv", [
    ([800, 333], 16, [1, 5, 16, 0], 16, 8), ([48], 16, [3], 16, 8), ([2000], 16, list(range(17)), 16, 8),
    ([1234], 7, [2, 7, 4], 8, 2), ([4300], 16, [1] * 40, 4, 2),
])
def test_attention_packed(lens, K, accepted, Hq, Hkv):
    vis = att.packed_visibility(K, accepted).tolist()
    _case(13 + K, [max(n, len(vis)) for n in lens], len(vis), Hq, Hkv, 16, 16, "packed", vis)


def test_attention_packed_odd_rows():
    """Rows that see nothing, only a second range, ranges that touch, overlap
    the first, are reversed or end past the context."""
    vis = [(0, 0, 0), (-500, 0, 0), (-500, 3, 9), (-400, -390, -380), (2, 2, 5), (3, 1, 6), (5, 9, 4), (1, 8, 5000),
           (5000, 0, 0), (-100, -90, 0)]
    _case(17, [410, 64], len(vis), 8, 2, 16, 16, "packed", vis)


def test_attention_ignores_what_a_row_does_not_see():
    """NaN codes and scales behind the context, in other pages and in table
    entries past it; a NaN key or value among the seen ones reaches the rows
    that see it and no other."""
    g = _gen(21)
    Q, H, P = 8, 2, 20
    nan = 0x7F
    for mode, vis in (("causal", None), ("full", None), ("packed", att.packed_visibility(2, [1, 0, 2]).tolist())):
        parts = [t.clone() for t in _like_data(g, P, H, 16, 16)]
        raw = [t.view(torch.uint8) for t in parts]
        table = torch.randperm(P, generator=g)[:16].view(1, 16).int()
        ctx = 150  # 9 pages and 6 tokens
        dead = [p for p in range(P) if p not in table[0, :10].tolist()]
        for t in raw[:2]:
            t[table[0, 9].long(), :, 6:] = nan
            t[dead] = nan
        for t in raw[2:]:
            t[dead] = 255
        q = torch.randn(1, Q, 4, D, generator=g).to(BF)
        far = table.clone()
        far[0, 10:] = torch.tensor([10 ** 6, -1, P, 2 ** 31 - 1, -2 ** 31, 0])
        clean = of.from_bytes(*parts)
        for tab in (table, far):
            out = _attend(q, _to_dev(parts), [ctx], tab, mode, vis)
            _close(out, *of.attention(q, clean, tab, [ctx], D ** -0.5, mode, vis))
            assert not out.isnan().any()
        # the block's own tokens: 142 .. 149
        for tok in (142, 144, 146, 149):
            for which in (0, 1):
                bad = [t.clone() for t in parts]
                bad[which].view(torch.uint8)[table[0, tok // 16].long(), 1, tok % 16, 37] = nan
                out = _attend(q, _to_dev(bad), [ctx], table, mode, vis)
                ref, wgt = of.attention(q, of.from_bytes(*bad), table, [ctx], D ** -0.5, mode, vis)
                _close(out, ref, wgt)


def test_attention_pages_outside_the_pool_read_as_zeros():
    g = _gen(23)
    parts = _like_data(g, 12, 2, 16, 16)
    table = torch.arange(12, dtype=torch.int32)[None].clone()
    table[0, 3], table[0, 7], table[0, 8] = -1, 12, 2 ** 31 - 1
    q = torch.randn(1, 16, 8, D, generator=g).to(BF)
    for ctx in (190, 120, 130):
        out = _attend(q, _to_dev(parts), [ctx], table, "causal")
        _close(out, *of.attention(q, of.from_bytes(*parts), table, [ctx], D ** -0.5))


def test_attention_contexts_past_their_bounds():
    """Lengths of zero and below, longer than the table, and a max_seqlen_k
    that is not a whole number of tiles."""
    g = _gen(29)
    parts = _like_data(g, 12, 2, 16, 16)
    table = torch.arange(12, dtype=torch.int32).view(3, 4)
    q = torch.randn(3, 4, 4, D, generator=g).to(BF)
    for mode in ("causal", "full"):
        out = _attend(q, _to_dev(parts), [0, -7, 1000], table, mode)
        _close(out, *of.attention(q, of.from_bytes(*parts), table, [0, -7, 1000], D ** -0.5, mode))
        assert not out[:2].any()
        out = _attend(q, _to_dev(parts), [33, 2, 37], table, mode, max_seqlen_k=37)
        _close(out, *of.attention(q, of.from_bytes(*parts), table, [33, 2, 37], D ** -0.5, mode))


def test_attention_arguments():
    g = _gen(31)
    parts = _like_data(g, 12, 2, 16, 16)
    cache, host = _to_dev(parts), of.from_bytes(*parts)
    table = torch.arange(12, dtype=torch.int32).view(2, 6)
    q = torch.randn(2, 4, 8, D, generator=g).to(BF)
    lens = torch.tensor([90, 33])
    want = of.attention(q, host, table, lens, 0.3)
    out = torch.empty(2, 4, 8, D, dtype=BF, device=DEV)
    wide = torch.randn(2, 8, 4, D, generator=g).to(BF).to(DEV)
    wide.copy_(q.transpose(1, 2))
    for qq, tab, ln in ((q.to(DEV), table, lens), (wide.transpose(1, 2), table.long(), lens.long())):
        got = fp8_kv.flash_attn_with_kvcache(qq, cache, ln.to(DEV), tab.to(DEV), softmax_scale=0.3, out=out)
        assert got is out
        _close(out, *want)
    full = fp8_kv.draft_block_attn(q.to(DEV), cache, lens.to(DEV), table.to(DEV), softmax_scale=0.3)
    _close(full, *of.attention(q, host, table, lens, 0.3, "full"))
    good = dict(q=q.to(DEV), cache=cache, cache_seqlens=lens.to(DEV), block_table=table.to(DEV))
    for bad in (dict(q=q[0].to(DEV)), dict(q=q[..., :64].to(DEV)), dict(q=q[:, :, :7].to(DEV)),
                dict(block_table=table[:1].to(DEV)), dict(cache_seqlens=lens[:1].to(DEV)), dict(max_seqlen_k=97),
                dict(max_seqlen_k=0), dict(out=out.float()), dict(out=out[:1]),
                dict(q=torch.zeros(2, 1, 130, D, dtype=BF, device=DEV)), dict(softmax_scale=0.0),
                dict(softmax_scale=-0.1), dict(softmax_scale=math.inf), dict(softmax_scale=math.nan)):
        with pytest.raises(ValueError):
            fp8_kv.flash_attn_with_kvcache(**{**good, **bad})
    vis = torch.tensor([[4, 0, 0]] * 4, dtype=torch.int32, device=DEV)
    for bad in (vis[:3], vis.long(), vis[:, :2]):
        with pytest.raises(ValueError):
            fp8_kv.packed_block_attn(q.to(DEV), cache, lens.to(DEV), table.to(DEV), bad)
    with pytest.raises(RuntimeError):
        fp8_kv.flash_attn_with_kvcache(q, cache, lens.to(DEV), table.to(DEV))


def test_attention_is_reproducible():
    g = _gen(37)
    parts = _like_data(g, 140, 4, 16, 16)
    cache = _to_dev(parts)
    table = torch.randperm(140, generator=g)[:130].view(1, 130).int()
    q = torch.randn(1, 16, 16, D, generator=g).to(BF)
    first = _attend(q, cache, [2075], table, "causal")
    for _ in range(5):
        assert torch.equal(_attend(q, cache, [2075], table, "causal"), first)


# -------------------------------------------------------------- all of it together
def _steps(cache, stream_of_inputs, table, Hq, Hkv):
    """Block after block as a layer runs them: append, then attention over what is held."""
    outs = []
    for qkv, pos, slots, lens, (qn, kn, inv) in stream_of_inputs:
        q = fp8_kv.qk_rope_append(qkv, pos, qn, kn, inv, cache, slots, Hq, Hkv, 1e-6)
        outs.append(fp8_kv.flash_attn_with_kvcache(q.view(table.shape[0], -1, Hq, D), cache, lens, table))
    return outs


def _session(seed, B=2, Hq=8, Hkv=2, page=16, starts=(0, 0)):
    """Prompts, single tokens and blocks with a rewind, over shuffled pages."""
    g = _gen(seed)
    width = 8
    table = torch.randperm(B * width + 3, generator=g)[: B * width].view(B, width).int()
    at, inputs = list(starts), []
    for n, back in ((40, 0), (1, 0), (16, 9), (16, 0), (1, 0), (5, 2), (3, 0)):
        qkv, qn, kn, inv = _rope_inputs(g, B * n, Hq, Hkv)
        pos = torch.cat([torch.arange(a, a + n) for a in at])
        row = torch.arange(B).repeat_interleave(n)
        slots = table[row, pos // page].long() * page + pos % page
        inputs.append((qkv.view(B * n, -1), pos, slots, torch.tensor([a + n for a in at], dtype=torch.int32),
                       (qn, kn, inv)))
        at = [a + n - back for a in at]
    return table, inputs


def _move(inputs):
    return [(a.to(DEV), b.to(DEV), c.to(DEV), d.to(DEV), tuple(x.to(DEV) for x in w)) for a, b, c, d, w in inputs]


def test_layer_steps_together():
    """Prefill, single tokens, blocks and rewinds against the oracle fed with
    the cache the kernels left before each step."""
    Hq, Hkv = 8, 2
    table, inputs = _session(41)
    cache = Fp8KV.empty(table.numel() + 3, 16, Hkv, DEV)
    for (qkv, pos, slots, lens, w), dev in zip(inputs, _move(inputs)):
        before = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
        q = fp8_kv.qk_rope_append(dev[0], dev[1], *dev[4], cache, dev[2], Hq, Hkv, 1e-6)
        _check_rope(q, cache, before, qkv.view(len(pos), -1, D), pos, *w, slots, Hq, Hkv, 1e-6)
        q4 = q.view(2, -1, Hq, D)
        out = fp8_kv.flash_attn_with_kvcache(q4, cache, dev[3], table.to(DEV))
        held = of.from_bytes(cache.k, cache.v, cache.k_scale, cache.v_scale)
        _close(out, *of.attention(q4.cpu(), held, table, lens, D ** -0.5))


def test_on_two_streams_at_once():
    """Two sessions on two streams, interleaved, give what each gives alone."""
    tables, dev, alone = [], [], []
    for seed in (43, 47):
        table, inputs = _session(seed)
        tables.append(table.to(DEV))
        dev.append(_move(inputs))
        alone.append(_steps(Fp8KV.empty(table.numel() + 3, 16, 2, DEV), dev[-1], tables[-1], 8, 2))
    torch.cuda.synchronize()
    for _ in range(3):
        caches = [Fp8KV.empty(t.numel() + 3, 16, 2, DEV) for t in tables]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = [[], []]
        for n in range(len(dev[0])):
            for i in (0, 1):
                with torch.cuda.stream(streams[i]):
                    outs[i] += _steps(caches[i], dev[i][n:n + 1], tables[i], 8, 2)
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], alone[i]))


def test_captured_and_replayed():
    """Two captured graphs of the same calls, replayed in turn with new inputs
    and eager work between, against eager results."""
    g = _gen(53)
    Hq, Hkv, B, Q = 16, 2, 2, 16
    table = torch.randperm(300, generator=g)[:280].view(B, 140).int().to(DEV)
    start = Fp8KV.empty(300, 16, Hkv, DEV)
    w = tuple(t.to(DEV) for t in _rope_inputs(g, 1, Hq, Hkv)[1:])
    k, v = (torch.randn(300 * 16, Hkv, D, generator=g).to(BF).to(DEV) for _ in range(2))
    fp8_kv.kv_append(k, v, start, torch.arange(300 * 16, device=DEV))

    def clone(c):
        return Fp8KV(*(t.view(torch.uint8).clone().view(t.dtype) for t in (c.k, c.v, c.k_scale, c.v_scale)))

    def fresh(seed):
        h = _gen(seed)
        n = 1000 + 37 * seed % 900
        pos = torch.arange(n, n + Q).repeat(B).to(DEV)
        row = torch.arange(B, device=DEV).repeat_interleave(Q)
        return (_rope_inputs(h, B * Q, Hq, Hkv)[0].view(B * Q, -1).to(DEV), pos,
                table[row, pos // 16].long() * 16 + pos % 16,
                torch.full((B,), n + Q, dtype=torch.int32, device=DEV))

    def step(cache, io):
        q = fp8_kv.qk_rope_append(io[0], io[1], *w, cache, io[2], Hq, Hkv, 1e-6)
        return fp8_kv.flash_attn_with_kvcache(q.view(B, Q, Hq, D), cache, io[3], table)

    graphs = []
    for _ in range(2):
        cache, io, owner = clone(start), fresh(0), []
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(clone(start), io)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with _lib.capture_workspaces(owner), torch.cuda.graph(graph):
            out = step(cache, io)
        graphs.append((graph, cache, io, out, owner))
    eager = [clone(start), clone(start)]
    for n in range(1, 7):
        i = n % 2
        graph, cache, io, out, _ = graphs[i]
        new = fresh(n)
        for a, b in zip(io, new):
            a.copy_(b)
        graph.replay()
        want = step(eager[i], new)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(cache.k.view(torch.uint8), eager[i].k.view(torch.uint8))
        assert torch.equal(cache.k_scale.view(torch.uint8), eager[i].k_scale.view(torch.uint8))
