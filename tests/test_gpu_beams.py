"""GPU: the operators together, as a search uses them: every row's keys and values are those of its own tokens after many
forks, and attention, selection and pages agree with their plain forms at every step; DecoderAttention over a 4-bit cache; the example."""
import importlib.util
import os

import pytest

import cache4_plain as plain
from conftest import ROOT
from helpers import say
from test_gpu_beam_select import check as check_selection
from test_gpu_cache4 import stored

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("beam_search", os.path.join(ROOT, "examples", "beam_search.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dt,W,Hq,Hkv,D,page,end", [("float16", 4, 8, 2, 64, 16, None), ("bfloat16", 3, 4, 1, 128, 32, 5), ("float16", 7, 3, 3, 96, 16, 3)])
def test_search(dev, dt, W, Hq, Hkv, D, page, end):
    """The key and value of a token depend on the token and its position, so that each row's cache can be told from its tokens."""
    import torch
    from forge_amd import ops
    from forge_amd.nn import PagedBeams
    say(f"search {dt} W={W} heads={Hq}/{Hkv} D={D} page={page}")
    d, V, B, steps = getattr(torch, dt), 40, 3, 24
    g = torch.Generator().manual_seed(D)
    table = torch.randn((2, V, Hkv, D), generator=g).to(dev)
    pos_part = torch.randn((2, 200, Hkv, D), generator=g).to(dev)

    def kv(tokens, positions):
        t, p = tokens.long().clamp_min(0), positions.long()
        return (table[0, t] + pos_part[0, p]).to(d), (table[1, t] + pos_part[1, p]).to(d)
    prompts = [torch.randint(V, (n,), generator=g).to(dev) for n in (page, 2, page * 2 - 1)]
    lens = [len(p) for p in prompts]
    beams = PagedBeams(B, W, 220, page, 140, dev)
    cache = torch.full(ops.cache4_shape(220, page, Hkv, D), 0xFF, dtype=torch.uint8, device=dev)
    slots = beams.start(lens)
    k, v = kv(torch.cat(prompts), torch.cat([torch.arange(n, device=dev) for n in lens]))
    ops.cache4_write(k, v, cache, slots)
    rows = [p.tolist() if w == 0 else None for p in prompts for w in range(W)]
    for step in range(steps):
        logits = (torch.randn((B, W, V), generator=g) * 2).to(d).to(dev)
        before, ended = beams.scores.clone(), beams.ended.clone()
        tokens, parents = beams.step(logits, [cache], end)
        check_selection(logits, before, W, (beams.scores, parents, tokens), None if end is None else ended, end or 0)
        par, tok = parents.tolist(), tokens.tolist()
        rows = [rows[b * W + par[b][w]] + [tok[b][w]] if par[b][w] >= 0 else None for b in range(B) for w in range(W)]
        live = [r for r, x in enumerate(rows) if x is not None]
        assert all(beams.slots[r] >= 0 for r in live) and beams.lens.tolist() == [len(x) - 1 if x else 0 for x in rows]
        k, v = kv(tokens.flatten(), beams.lens)
        ops.cache4_write(k, v, cache, beams.slots)
        q = torch.randn((B * W, 1, Hq, D), generator=g).to(d).to(dev)
        out = ops.cache4_attention(q, cache, beams.table, beams.lens)
        names = torch.bincount(beams.table[beams.table >= 0].long(), minlength=220)
        assert torch.equal(names.to(torch.int32), beams.refs)
        for r in live:
            n = len(rows[r])
            at = torch.arange(n, device=dev)
            mine = (beams.table[r, at // page].long() * page + at % page).to(torch.int32)
            wk, wv = kv(torch.tensor(rows[r], device=dev), at)
            rk, rv = ops.cache4_read(cache, mine, D, d)
            assert torch.equal(rk, stored(wk, D, dt)) and torch.equal(rv, stored(wv, D, dt)), (step, r)
            if step % 6 == 0 or r == live[-1]:
                hk, hv = plain.held(wk), plain.held(wv)
                for h in range(Hq):
                    a, b = ([t[:, h // (Hq // Hkv)] for t in x] for x in (hk, hv))
                    plain.check(out[r, :, h], q[r, :, h], a, b, torch.ones((1, n), dtype=torch.bool, device=dev), D ** -0.5)


@pytest.mark.parametrize("dt,D,T", [("float16", 64, 1), ("bfloat16", 128, 6), ("float16", 96, 3)])
def test_decoder_attention(dev, dt, D, T):
    """DecoderAttention over a 4-bit cache is its own operators, called one by one."""
    import torch
    from forge_amd import ops
    from forge_amd.nn import DecoderAttention
    say(f"DecoderAttention over 4 bits {dt} D={D} T={T}")
    d = getattr(torch, dt)
    torch.manual_seed(D)
    block = DecoderAttention(256, 6, 2, D, 300, 32, dtype=d).to(dev)
    for layer in (block.qkv, block.out):
        layer.quantize_weight(torch.randn((layer.out_features, layer.in_features), device=dev) * layer.in_features ** -0.5)
    lens, page = [20, 1, 75], 16
    width = (max(lens) + T + page - 1) // page
    table = torch.randperm(3 * width, generator=torch.Generator().manual_seed(1)).view(3, width).to(torch.int32).to(dev)
    caches = [torch.zeros(ops.cache4_shape(3 * width, page, 2, D), dtype=torch.uint8, device=dev) for _ in range(2)]

    def rows(first, n):
        pos = [torch.arange(f, f + m, device=dev) for f, m in zip(first, n)]
        slots = [table[b, p // page].long() * page + p % page for b, p in enumerate(pos)]
        return torch.cat(pos).to(torch.int32), torch.cat(slots).to(torch.int32)
    pos, slots = rows([0] * 3, lens)
    cu = torch.tensor([0, 20, 21, 96], dtype=torch.int32, device=dev)
    x = torch.randn((96, 256), device=dev).to(d)
    got = block.prompt(x, cu, pos, caches[0], None, slots)
    q, k, v = block._heads(x)
    q, k = ops.qk_norm_rope(q, k, block.q_norm, block.k_norm, block.cos, block.sin, pos, eps=block.eps)
    ops.cache4_write(k, v, caches[1], slots)
    assert torch.equal(got, block.out(ops.prompt_attention(q, k, v, cu).view(96, -1)))
    assert torch.equal(caches[0], caches[1])
    x = torch.randn((3, T, 256), device=dev).to(d)
    pos, slots = rows(lens, [T] * 3)
    clens = torch.tensor(lens, dtype=torch.int32, device=dev)
    tree = torch.ones((3, T), dtype=torch.int64, device=dev) if T > 1 else None
    got = block.cached(x, pos, caches[0], None, slots, table, clens, tree)
    q, k, v = block._heads(x.view(3 * T, 256))
    q, k = ops.qk_norm_rope(q, k, block.q_norm, block.k_norm, block.cos, block.sin, pos, eps=block.eps)
    ops.cache4_write(k, v, caches[1], slots)
    o = ops.cache4_attention(q.view(3, T, 6, D), caches[1], table, clens, tree)
    assert torch.equal(got, block.out(o.view(3, T, -1)))


def test_example(dev, example):
    """The example runs; its beams are in order, and finite."""
    import torch
    found, scores, worst = example.main()
    assert found.shape == (3, 4, 12) and torch.isfinite(scores).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    assert worst < float("inf") and (found >= 0).all()
