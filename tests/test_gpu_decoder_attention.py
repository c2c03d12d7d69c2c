"""GPU: Int4Linear and DecoderAttention, and the example that runs them over prompts, single tokens and drafts,
against the block in 64 bits.

Bound of a whole block: each of its four 16-bit roundings (projection, rotation, attention weights, attention) moves a
value by u of its size, and the output projection sums them; 8 u of the largest output is far above
their sum in the 2-norm and far below a wrong key, mask or position (differences of the outputs' own size)."""
import importlib.util
import os

import pytest

from conftest import ROOT
from helpers import say
from test_gpu_int4 import check, unpack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decoder_attention", os.path.join(ROOT, "examples", "decoder_attention.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dt,bias,G", [("float16", True, 128), ("bfloat16", False, 32)])
def test_int4_linear_module(dev, dt, bias, G):
    import torch
    from forge_amd.nn import Int4Linear
    K, N = 384, 50
    layer = Int4Linear(K, N, bias, G, getattr(torch, dt)).to(dev)
    x = torch.randn((2, 3, K), device=dev).to(getattr(torch, dt))
    assert (layer(x) == 0).all()                          # as made, all weights are zero
    w = torch.randn((N, K), device=dev) * 0.05
    layer.quantize_weight(w)
    if bias:
        with torch.no_grad():
            layer.bias.copy_(torch.randn(N))
    y = layer(x)
    assert y.shape == (2, 3, N)
    check(y.view(6, N), x.view(6, K), unpack(layer.w_int4, K), layer.w_scale, layer.bias, G)
    other = Int4Linear(K, N, bias, G, getattr(torch, dt)).to(dev)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    with pytest.raises(NotImplementedError):
        layer(x.requires_grad_(True)).sum().backward()
    with pytest.raises(ValueError):
        Int4Linear(100, 8)
    with pytest.raises(TypeError):
        Int4Linear(128, 8, dtype=torch.float32)


def plain_block(block, x, seen, positions):
    """The block in 64 bits over tokens x (n, hidden) with the mask seen (n, n)."""
    import torch

    def linear(layer, x):
        q = unpack(layer.w_int4, layer.in_features).to(x.device).double()
        return x @ (q * layer.w_scale.double().repeat_interleave(layer.group_size, 1)).T
    D, H, Hk = block.head_dim, block.heads, block.kv_heads
    q, k, v = linear(block.qkv, x.double()).view(len(x), -1, D).split((H, Hk, Hk), 1)

    def norm_rope(t, w):
        t = t / (t.square().mean(-1, keepdim=True) + block.eps).sqrt() * w.double()
        c, s = block.cos[positions].double()[:, None], block.sin[positions].double()[:, None]
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    q, k = norm_rope(q, block.q_norm), norm_rope(k, block.k_norm)
    o = torch.empty_like(q)
    for h in range(H):
        z = (q[:, h] @ k[:, h // (H // Hk)].T) * D ** -0.5
        o[:, h] = torch.softmax(z.masked_fill(~seen, float("-inf")), -1) @ v[:, h // (H // Hk)]
    return linear(block.out, o.flatten(1))


@pytest.mark.parametrize("dt,heads,kv,D", [("float16", 8, 2, 64), ("bfloat16", 6, 6, 128), ("float16", 4, 1, 80)])
def test_prompts_tokens_and_drafts(dev, example, dt, heads, kv, D):
    import torch
    u = 2.0 ** -11 if dt == "float16" else 2.0 ** -8
    block = example.make(dev, getattr(torch, dt), 256, heads, kv, D, 32 if D == 80 else 64, seed=D)
    lens, steps = [20, 1, 75], 3
    parents = torch.tensor([[-1, -1, 0, 1, 2, 2], [-1, 0, 1, 2, 3, 4], [-1, 0, 0, 0, -1, 4]])
    x = [torch.randn((n + steps + 6, 256), device=dev).to(getattr(torch, dt)) for n in lens]
    say(f"decoder attention {dt} heads={heads}/{kv} D={D}")
    prompt, single, drafts = example.run(block, x, lens, steps, parents, dev)
    start = 0
    for b, n in enumerate(lens):
        N = n + steps + 6
        seen = torch.ones((N, N), dtype=torch.bool, device=dev).tril()
        pos = torch.arange(N, device=dev)
        seen[n + steps:, n + steps:] = False
        for t in range(6):
            p, depth = t, -1
            while p >= 0:
                seen[n + steps + t, n + steps + p] = True
                p, depth = int(parents[b, p]), depth + 1
            pos[n + steps + t] = n + steps + depth
        want = plain_block(block, x[b], seen, pos)
        got = torch.cat([prompt[start:start + n], single[b], drafts[b]])
        start += n
        err = (got.double() - want).abs().max().item()
        assert err <= 8 * u * want.abs().max().item(), (b, err)


def test_example(dev, example):
    """Each phase agrees with the whole sequence at once to the same bound (twice: both sides are rounded)."""
    worst = example.main()
    assert max(worst) <= 2 * 8 * 2.0 ** -11 * 8.0
