"""The 64-bit oracle of the 8-bit cache against torch's own conversions (CPU),
and what the cache object refuses."""
from __future__ import annotations

import math

import pytest
import torch

from d3d_amd.fp8_kv import Fp8KV
from oracle import fp8_kv as of


def test_round_e4m3_is_torchs():
    g = torch.Generator().manual_seed(1)
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(of.round_e4m3(codes)[~codes.isnan()], codes[~codes.isnan()])
    mid = codes[codes >= 0].sort().values[:-1]
    ties = (mid[1:] + mid[:-1]) / 2
    x = torch.cat([ties, -ties, torch.randn(4096, generator=g).double() * 40, torch.rand(4096, generator=g).double() / 64])
    x = x.float()
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(of.round_e4m3(x.double()), want)
    assert of.round_e4m3(torch.tensor([math.inf, -math.inf, math.nan], dtype=torch.float64)).isnan().all()


def test_need_exp_is_the_least():
    for amax in (1e-30, 0.1, 1.0, 448.0, math.nextafter(448.0, 500), 447.9, 3.0e38, 2.0 ** -100, 1.75, 1.7500001):
        e = of.need_exp(amax)
        if of.E_MIN < e < of.E_MAX:
            assert amax <= 448 * 2.0 ** e and amax > 448 * 2.0 ** (e - 1)
    assert of.need_exp(0.0) == of.E_MIN and of.need_exp(2.0 ** -120) == of.E_MIN and of.need_exp(1e300) == of.E_MAX


def test_growing_a_block_keeps_normal_codes():
    """Token by token, with each larger than the last, gives what one call gives."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(16, 1, 128, generator=g).double() * torch.exp2(torch.arange(16.0) / 4).double()[:, None, None]
    x = torch.where(x.abs() < 2.0 ** -4, 2.0 ** -4, x)  # within 2^-14 of the block's largest
    step = one = of.empty(1, 1, 16, 16)
    for n in range(16):
        step = of.append(step, x[n:n + 1], x[n:n + 1], [n])
    one = of.append(one, x, x, list(range(16)))
    assert torch.equal(step["k_exp"], one["k_exp"]) and torch.equal(step["k"], one["k"])


def _parts(P=2, H=1, page=16, blocks=1, D=128):
    c = [torch.zeros(P, H, page, D, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    s = [torch.zeros(P, H, blocks, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    return c + s


@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 64), (256, 256), (48, 16), (96, 32)])
def test_cache_shapes(page, block):
    c = Fp8KV.empty(3, page, 2, "cpu", block=block)
    assert (c.num_pages, c.kv_heads, c.page_size, c.block) == (3, 2, page, block)
    k, v = c.dequantize()
    assert k.shape == (3, page, 2, 128) and k.dtype == torch.bfloat16 and not v.any()


@pytest.mark.parametrize("page,block", [(8, 8), (16, 8), (24, 16), (512, 512), (48, 48), (16, 0), (16, 32)])
def test_cache_refuses_blocks(page, block):
    with pytest.raises(ValueError):
        Fp8KV.empty(3, page, 2, "cpu", block=block)


def test_cache_refuses_parts():
    c = _parts()
    Fp8KV(*c)
    with pytest.raises(ValueError, match="equal shape"):
        Fp8KV(c[0], c[1][:1], c[2], c[3])
    with pytest.raises(ValueError, match="equal shape"):
        Fp8KV(c[0], c[1], c[2], c[3][:1])
    with pytest.raises(ValueError, match="e4m3"):
        Fp8KV(c[0].view(torch.uint8), c[1], c[2], c[3])
    with pytest.raises(ValueError, match="e8m0"):
        Fp8KV(c[0], c[1], c[2].view(torch.uint8), c[3])
    with pytest.raises(ValueError, match="128"):
        Fp8KV(*_parts(D=64))
    with pytest.raises(ValueError, match="contiguous"):
        d = _parts(P=4)
        Fp8KV(d[0][::2], d[1][::2], d[2][::2], d[3][::2])
    with pytest.raises(ValueError, match="aligned"):
        raw = torch.zeros(2 * 16 * 128 + 16, dtype=torch.uint8)
        at = (-raw.data_ptr()) % 16 + 8
        Fp8KV(raw[at:at + 2 * 16 * 128].view(torch.float8_e4m3fn).view(2, 1, 16, 128), c[1], c[2], c[3])
    with pytest.raises(ValueError, match="at least one"):
        Fp8KV(*_parts(P=0))


def test_no_cpu_path():
    from d3d_amd import fp8_kv
    c = Fp8KV.empty(1, 16, 1, "cpu")
    x = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp8_kv.kv_append(x, x, c, torch.zeros(1, dtype=torch.int64))


@pytest.mark.parametrize("change,expect", [
    (dict(), -4), (dict(T=-1), -1), (dict(H=0), -1), (dict(D=64), -5), (dict(page=0), -1), (dict(pages=0), -1),
    (dict(block=8), -5), (dict(block=512, page=512), -5), (dict(block=24, page=48), -5), (dict(block=32), -5),
    (dict(T=0), 0),
])
def test_append_refusals_without_launching(d3d_lib, change, expect):
    a = dict(T=4, H=2, D=128, page=16, block=16, pages=3) | change
    st = d3d_lib.d3d_kv_append_fp8(None, None, 256, 256, None, None, None, None, None, a["T"], a["H"], a["D"],
                                   a["page"], a["block"], a["pages"], None)
    assert st == expect
    st = d3d_lib.d3d_qk_rope_append_fp8(None, None, None, None, None, None, None, None, None, None, None, a["T"], 4,
                                        a["H"], a["D"], 1e-6, a["page"], a["block"], a["pages"], None)
    assert st == expect


def test_append_refuses_unaligned_rows(d3d_lib):
    """Pointers are checked on the host: none of these is read."""
    def call(k=4096, stride=256, kc=4096):
        return d3d_lib.d3d_kv_append_fp8(k, 4096, stride, 256, kc, 4096, 4096, 4096, 4096, 1, 2, 128, 16, 16, 1, None)
    assert call(k=4100) == -5 and call(stride=258) == -5 and call(stride=-256) == -5 and call(kc=4104) == -5


@pytest.mark.parametrize("change,expect", [
    (dict(), -4), (dict(B=0), -1), (dict(B=65536), -1), (dict(Q=0), -1), (dict(Hq=7), -1), (dict(D=64), -5),
    (dict(Hq=130, Hkv=2), -5), (dict(block=8), -5), (dict(block=32), -5), (dict(ctx=0), -1), (dict(ctx=33), -1),
    (dict(max_pages=0), -1), (dict(pages=0), -1),
])
def test_attention_refusals_without_launching(d3d_lib, change, expect):
    a = dict(B=1, Q=4, Hq=4, Hkv=2, D=128, page=16, block=16, max_pages=2, pages=2, ctx=32) | change
    tail = (a["B"], a["Q"], a["Hq"], a["Hkv"], a["D"], a["page"], a["block"], a["max_pages"], a["pages"], 1.0,
            a["ctx"], None, 0, None)
    assert d3d_lib.d3d_verify_attn_paged_fp8(*[None] * 8, *tail) == expect
    assert d3d_lib.d3d_draft_block_attn_fp8(*[None] * 8, *tail) == expect
    assert d3d_lib.d3d_packed_block_attn_fp8(*[None] * 9, *tail) == expect
