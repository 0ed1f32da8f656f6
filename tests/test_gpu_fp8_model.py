"""The models, the runner and the engine over the 8-bit cache (GPU).

The attention calls of a forward are recorded and done again by the bf16
attention over the same cache's values (a bf16 holds them exactly): each side
is off by half a bf16 step, 2^-8 of the output, and 2^-8 + 2^-10 of sum p |v| /
sum p for its rounded probabilities and fp32 sums, as the kernels' own tests
derive, and sum p |v| / sum p is at most the largest |v| of the head.
"""
from __future__ import annotations

import pytest
import torch

from d3d_amd import attention as att
from d3d_amd import fp8_kv
from d3d_amd.engine import Engine, generate_ar
from d3d_amd.model import (ModelShape, PagedKV, Qwen3PagedModel, Sequence, block_inputs, prefill, release, reserve)
from oracle import fp8_kv as of

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TARGET = ModelShape(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=128, mlp=512, vocab=1000)
DRAFT = ModelShape(layers=1, hidden=256, heads=4, kv_heads=2, head_dim=128, mlp=256, vocab=1000)


def _prompts(seed, lens):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 999, (n,), generator=g).tolist() for n in lens]


def _block(model, kv, seqs, Q, causal, vis=None):
    for s in seqs:
        reserve(kv, s, "m", s.prefix + Q)
    tables, slots, lens, logical, mx = block_inputs(kv, seqs, "m", [s.prefix for s in seqs], Q, DEV)
    ids = torch.arange(len(seqs) * Q, device=DEV).view(len(seqs), Q) % 999
    return model(ids, logical, kv, tables, lens, slots, causal=causal, max_context=mx, q_vis=vis)


@pytest.mark.parametrize("kind", ["verify", "draft", "packed"])
def test_forward_attends_over_the_cache(kind, monkeypatch):
    draft = kind != "verify"
    model = Qwen3PagedModel(TARGET, DEV, draft=draft, seed=3, init_std=0.05)
    kv = PagedKV(TARGET, 64, 16, DEV, kv_dtype="fp8")
    calls = []
    for name in ("flash_attn_with_kvcache", "packed_block_attn"):
        real = getattr(fp8_kv, name)

        def record(q, cache, lens, table, *rest, real=real, name=name, **kw):
            out = real(q, cache, lens, table, *rest, **kw)
            calls.append((name, q.clone(), cache.dequantize(), lens.clone(), table.clone(), rest, kw, out.clone()))
            return out

        monkeypatch.setattr(fp8_kv, name, record)
    seqs = [Sequence(i, p) for i, p in enumerate(_prompts(1, [37, 5, 90]))]
    prefill(model, kv, seqs, "m")
    if kind == "packed":
        vis = att.packed_visibility(16, [3, 16, 0]).to(DEV)
        _block(model, kv, seqs, 64, False, vis)
    else:
        _block(model, kv, seqs, 16, kind == "verify")
    assert len(calls) == 2 * TARGET.layers
    for name, q, (k, v), lens, table, rest, kw, out in calls:
        want = getattr(att, name)(q, k, v, lens, table, *rest, **kw).double()
        got = out.double()
        top = v.double().abs().amax((0, 1, 3)).repeat_interleave(TARGET.heads // TARGET.kv_heads)[None, None, :, None]
        tol = 2 * (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * top)
        assert bool(((got - want).abs() <= tol).all())
        assert float((got - want).norm() / want.norm()) <= 2 * (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -10)


def test_cache_holds_the_bf16_caches_values():
    """The first layer's input is the same for both caches: its values are the
    codes of the bf16 cache's, its keys within half a code and the bf16 path's
    own roundings (two before and one after the rotation, each at most 2^-9 of
    the pair's length, which is at most sqrt(2) of the row's largest |x|)."""
    seqs_of = lambda: [Sequence(i, p) for i, p in enumerate(_prompts(2, [50, 16, 33]))]  # noqa: E731
    model = Qwen3PagedModel(TARGET, DEV, draft=False, seed=5, init_std=0.05)
    kvs = [PagedKV(TARGET, 32, 16, DEV), PagedKV(TARGET, 32, 16, DEV, kv_dtype="fp8")]
    for kv in kvs:
        prefill(model, kv, seqs_of(), "m")
    used = [p for n in (50, 16, 33) for p in range(-(-n // 16))]  # pages are handed out in order
    tokens = [s for base, n in ((0, 50), (64, 16), (80, 33)) for s in range(base, base + n)]
    assert len(used) == 8
    k, v = (t[0].cpu().double().view(-1, 2, 128)[tokens] for t in (kvs[0].k, kvs[0].v))
    want = of.append(of.empty(32, 2, 16, 16), k, v, tokens)
    got = of.from_bytes(kvs[1].fp8[0].k, kvs[1].fp8[0].v, kvs[1].fp8[0].k_scale, kvs[1].fp8[0].v_scale)
    assert torch.equal(got["v"], want["v"]) and torch.equal(got["v_exp"], want["v_exp"])
    pg, sl = torch.tensor(tokens) // 16, torch.tensor(tokens) % 16
    held = of.values(got)[0][pg, :, sl]
    scale = torch.exp2(got["k_exp"].double())[pg, :, 0][..., None]
    row = k.abs().amax(-1, keepdim=True)
    tol = torch.maximum(2.0 ** -4 * k.abs(), 2.0 ** -10 * scale) + 3 * 2.0 ** -9 * 2 ** 0.5 * (1 + 2.0 ** -4) * row
    assert bool(((held - k).abs() <= tol).all())


def test_cache_arguments():
    with pytest.raises(ValueError, match="kv_dtype"):
        PagedKV(TARGET, 4, 16, DEV, kv_dtype="int8")
    with pytest.raises(ValueError, match="head dimension"):
        PagedKV(ModelShape(layers=1, hidden=64, heads=1, kv_heads=1, head_dim=64, mlp=64), 4, 16, DEV, kv_dtype="fp8")
    with pytest.raises(ValueError, match="block"):
        PagedKV(TARGET, 4, 8, DEV, kv_dtype="fp8")
    assert PagedKV(TARGET, 4, 64, DEV, kv_dtype="fp8", scale_block=32).fp8[1].block == 32


def _engine(seed, **kw):
    eng = Engine(TARGET, DRAFT, pages=16, seed=seed, mask_id=999, kv_dtype="fp8", **kw)
    for r in (eng.target, eng.draft):
        r.model.lm_head.mul_(20.0)
    return eng


def test_engine_graphs_match_eager_and_pages_come_back():
    """Replayed steps give the eager run's tokens, a second run over used pages
    gives the first one's, and no page is lost."""
    outs = []
    for graphs in (False, True):
        eng = _engine(11, use_graphs=graphs)
        prompts = _prompts(4, [48, 17, 30])
        for _ in range(2):
            res = eng.generate(prompts, 3, max_new_tokens=30, ignore_eos=True)
            assert [len(o["tokens"]) for o in res["outputs"]] == [30] * 3
            assert res["target_free_pages"] == eng.target.kv.num_pages
            outs.append([o["tokens"] for o in res["outputs"]])
    assert all(o == outs[0] for o in outs)


def test_target_only_decoding_runs_single_tokens():
    """One token per request and forward: the first tokens are those that one
    forward over the same prompts gives, and runs repeat."""
    eng = _engine(17)
    prompts = _prompts(6, [20, 45])
    first = eng.target.prefill([Sequence(i, p) for i, p in enumerate(prompts)])
    runs = [[o["tokens"] for o in generate_ar(eng.target, prompts, 2, 20, ignore_eos=True)["outputs"]] for _ in range(2)]
    assert runs[0] == runs[1] and [t[0] for t in runs[0]] == first
