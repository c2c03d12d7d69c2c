"""GPU: prompt_attention against the plain 64-bit form, within the bound of attention_plain.py."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu


def make(lens, Hq, Hkv, D, dt, dev, seed, tail=0):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens) + tail
    d = getattr(torch, dt)
    q = (torch.randn((T, Hq, D), generator=g, device=dev) * 1.5).to(d)
    kv = (torch.randn((T, 2 * Hkv, D), generator=g, device=dev) * 1.5).to(d)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return q, kv[:, :Hkv], kv[:, Hkv:], torch.tensor(cu, dtype=torch.int32, device=dev)


def check_all(out, q, k, v, lens, causal, scale=None):
    import torch
    from attention_plain import check
    at, group = 0, q.shape[1] // k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for n in lens:
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        seen = i[None] <= i[:, None] if causal else torch.ones((n, n), dtype=torch.bool, device=q.device)
        for h in range(q.shape[1]):
            check(out[at:at + n, h], q[at:at + n, h], k[at:at + n, h // group], v[at:at + n, h // group], seen, scale)
        at += n
    assert (out[at:] == 0).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([1], 1, 1, 8), ([2, 0, 1], 2, 1, 64), ([31, 32, 33], 4, 2, 64), ([63, 64, 65], 2, 2, 80), ([127, 1, 129], 3, 1, 96),
    ([200], 8, 1, 128), ([0, 0, 257, 0], 4, 4, 128), ([300, 70], 2, 2, 200), ([130], 6, 3, 256), ([515, 1, 1, 1, 258], 2, 1, 128),
    ([1] * 40, 2, 2, 64), ([700], 9, 9, 72)])
def test_prompt_attention(dev, lens, Hq, Hkv, D, causal, dt):
    from forge_amd import ops
    q, k, v, cu = make(lens, Hq, Hkv, D, dt, dev, sum(lens) + D)
    say(f"prompt_attention {dt} lens={lens} Hq={Hq} Hkv={Hkv} D={D} causal={causal}")
    check_all(ops.prompt_attention(q, k, v, cu, causal=causal), q, k, v, lens, causal)


@pytest.mark.parametrize("tokens,Hq,Hkv", [(2100, 8, 2), (1500, 32, 8), (4500, 4, 1)])
def test_long(dev, tokens, Hq, Hkv):
    """Sizes that take the widest workgroups."""
    from forge_amd import ops
    q, k, v, cu = make([tokens, 77], Hq, Hkv, 128, "float16", dev, tokens)
    say(f"prompt_attention tokens={tokens} Hq={Hq}")
    check_all(ops.prompt_attention(q, k, v, cu), q, k, v, [tokens, 77], True)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [([900], 32, 8, 64), ([901, 30], 32, 32, 80), ([450], 3, 1, 256), ([260], 2, 2, 48),
                                           ([641, 2], 5, 5, 128)])
def test_many_tiles(dev, lens, Hq, Hkv, D, causal, dt):
    """Chains of tiles longer than the buffers, at every head size and both ways of sharing the keys."""
    from forge_amd import ops
    q, k, v, cu = make(lens, Hq, Hkv, D, dt, dev, sum(lens) + D)
    say(f"prompt_attention {dt} lens={lens} Hq={Hq} Hkv={Hkv} D={D} causal={causal}")
    check_all(ops.prompt_attention(q, k, v, cu, causal=causal), q, k, v, lens, causal)


def test_scale_tail_and_growing_scores(dev):
    """A scale of the caller's, tokens after the last sequence, and scores whose maximum keeps growing along
    the keys (the sums are rescaled again and again) or falls from the first on."""
    import torch
    from forge_amd import ops
    lens = [400, 90]
    q, k, v, cu = make(lens, 2, 1, 64, "float16", dev, 3, tail=37)
    out = torch.full_like(q, 5.0)
    assert ops.prompt_attention(q, k, v, cu, scale=0.5, out=out) is out
    check_all(out, q, k, v, lens, True, 0.5)
    for sign in (1.0, -1.0):
        k2 = k.clone()
        k2[:400, 0] = q[:400].mean(1) * 0.1 + sign * torch.linspace(0, 3, 400, device=dev).half()[:, None]
        q2 = q.abs()
        for causal in (True, False):
            check_all(ops.prompt_attention(q2, k2, v, cu, causal=causal), q2, k2, v, lens, causal)


@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
def test_masked_places_hold_anything(dev, D, dt):
    """Infinities and NaN in keys and values that a row does not see (later in its sequence, in the
    neighbouring sequences, after the last one) do not touch it; rows that see them are not finite."""
    import torch
    from forge_amd import ops
    lens = [70, 100, 40]
    q, k, v, cu = make(lens, 4, 2, D, dt, dev, D, tail=9)
    k, v = k.clone(), v.clone()
    k[:70] = float("nan")
    v[:70] = float("inf")
    k[170:], v[170:] = float("inf"), float("nan")
    v[70 + 60, 0, 3] = float("nan")
    v[70 + 97, 1, 5] = float("-inf")
    out = ops.prompt_attention(q, k, v, cu)
    from attention_plain import check
    i = torch.arange(100, device=dev)
    seen = i[None] <= i[:, None]
    mid = out[70:170]
    for h in range(4):
        g = h // 2
        until = 60 if g == 0 else 97
        check(mid[:until, h], q[70:70 + until, h], k[70:170, g], v[70:170, g], seen[:until], D ** -0.5)
        bad = 3 if g == 0 else 5
        assert not torch.isfinite(mid[until:, h, bad]).any()
        rest = [d for d in range(D) if d != bad]
        check(mid[:, h][:, rest], q[70:170, h], k[70:170, g], v[70:170, g][:, rest], seen, D ** -0.5)
    # values of masked keys at the type's extremes
    v[70:170] = torch.finfo(v.dtype).max
    v[70:100] = 1.0
    out = ops.prompt_attention(q, k, v, cu)
    assert torch.allclose(out[70:100].float(), torch.ones((), device=dev), rtol=2 * 2.0 ** -8, atol=0)


def test_infinite_scores(dev):
    """A key of minus infinity against a positive query weighs nothing; plus infinity gives NaN, as exp(inf - inf)."""
    import torch
    from forge_amd import ops
    q, k, v, cu = make([40], 1, 1, 64, "bfloat16", dev, 9)
    q, k = q.abs() + 0.1, k.clone()
    k[5, 0, 7] = float("-inf")
    out = ops.prompt_attention(q, k, v, cu)
    from attention_plain import check
    i = torch.arange(40, device=dev)
    seen = i[None] <= i[:, None]
    seen[:, 5] = False
    rows = [r for r in range(40) if r != 5]
    check(out[rows, 0], q[rows, 0], k[:, 0], v[:, 0], seen[rows], 0.125)
    k[5, 0, 7] = float("inf")
    out = ops.prompt_attention(q, k, v, cu)
    assert torch.isnan(out[5:]).all() and torch.isfinite(out[:5]).all()


def test_strides(dev):
    """Heads in any order of tokens and heads, a KV head shared by expansion, and offsets past 32 bits."""
    import torch
    from forge_amd import ops
    q, k, v, cu = make([150], 4, 4, 64, "float16", dev, 10)
    want = ops.prompt_attention(q, k, v, cu)
    qh, kh, vh = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))    # head-major memory
    assert torch.equal(ops.prompt_attention(qh, kh, vh, cu), want)
    k1, v1 = k[:, :1].expand(150, 4, 64), v[:, :1].expand(150, 4, 64)
    assert torch.equal(ops.prompt_attention(q, k1, v1, cu), ops.prompt_attention(q, k[:, :1], v[:, :1], cu))
    step = 1 << 23                                                    # 16 MB from token to token, 2.5 GB in all
    big = torch.empty(((150 - 1) * step + 64,), dtype=torch.float16, device=dev)
    far = big.as_strided((150, 1, 64), (step, 64, 1))
    for put in ("k", "v", "q"):
        src = {"k": k, "v": v, "q": q}[put][:, :1]
        far.copy_(src)
        args = {"q": q[:, :1], "k": k[:, :1], "v": v[:, :1]}
        args[put] = far
        assert torch.equal(ops.prompt_attention(args["q"], args["k"], args["v"], cu),
                           ops.prompt_attention(q[:, :1], k[:, :1], v[:, :1], cu))


def test_boundaries_outside_the_tokens(dev):
    """Boundaries past the tokens or falling are kept inside the buffers; sequences that they leave whole are right."""
    import torch
    from forge_amd import ops
    q, k, v, _ = make([100], 1, 1, 64, "float16", dev, 11)
    cu = torch.tensor([0, 60, 1000], dtype=torch.int32, device=dev)
    check_all(ops.prompt_attention(q, k, v, cu), q, k, v, [60, 40], True)
    cu = torch.tensor([0, 100, 50, 100], dtype=torch.int32, device=dev)
    assert ops.prompt_attention(q, k, v, cu).shape == q.shape


def test_graph_and_stream(dev):
    import torch
    from forge_amd import ops
    q, k, v, cu = make([90, 200], 4, 2, 128, "bfloat16", dev, 12)
    want = ops.prompt_attention(q, k, v, cu)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_attention(q, k, v, cu, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, cu, out=out)
    for i in range(3):
        q.mul_(0.5)
        want = ops.prompt_attention(q, k, v, cu)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(dev):
    import torch
    from forge_amd import ops
    q, k, v, cu = make([20], 4, 2, 64, "float16", dev, 13)
    f = ops.prompt_attention
    for bad in (lambda: f(q.float(), k, v, cu), lambda: f(q, k.to(torch.bfloat16), v, cu), lambda: f(q, k, v, cu.long())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: f(q[:, :3], k, v, cu), lambda: f(q, k, v[:, :1], cu), lambda: f(q[..., :60], k[..., :60], v[..., :60], cu),
                lambda: f(q, k[:10], v[:10], cu), lambda: f(q, k, v, cu[:1]), lambda: f(q, k, v, cu.cpu()),
                lambda: f(q[..., 4:44], k[..., 4:44], v[..., 4:44], cu), lambda: f(q, k, v, cu, scale=-1.0),
                lambda: f(q, k, v, cu, scale=0.0), lambda: f(q, k, v, cu, scale=float("nan")),
                lambda: f(q, k, v, cu, out=q[:, :2]), lambda: f(q, k[..., :32], v[..., :32], cu)):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros((2, 1, 264), dtype=torch.float16, device=dev)
    with pytest.raises(ValueError):
        f(wide, wide, wide, cu)
    assert f(q[:0], k[:0], v[:0], cu).shape == (0, 4, 64)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([1025], 4, 2, 64), ([300, 0, 1, 31], 3, 1, 40), ([1100, 33], 4, 4, 80), ([257], 1, 1, 96), ([997, 5], 4, 1, 128),
    ([400, 260, 3], 6, 2, 128), ([1030], 10, 5, 64), ([1030], 12, 4, 128), ([1500], 9, 3, 80), ([901, 64], 4, 2, 256),
    ([1, 290], 8, 8, 200), ([650], 32, 8, 136)])
def test_few_workgroups(dev, lens, Hq, Hkv, D, causal, dt):
    """Sizes that leave CUs over, whose workgroups take fewer rows (up to 128 values a head)."""
    from forge_amd import ops
    q, k, v, cu = make(lens, Hq, Hkv, D, dt, dev, sum(lens) + D)
    say(f"prompt_attention {dt} lens={lens} Hq={Hq} Hkv={Hkv} D={D} causal={causal}")
    check_all(ops.prompt_attention(q, k, v, cu, causal=causal), q, k, v, lens, causal)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_workgroups_masked_places(dev, D):
    """NaN and infinities after a row and in the next sequence, with waves that share rows."""
    import torch
    from attention_plain import check
    from forge_amd import ops
    lens = [290, 40]
    q, k, v, cu = make(lens, 2, 1, D, "float16", dev, D + 1)
    k, v = k.clone(), v.clone()
    k[290:], v[290:] = float("nan"), float("inf")
    v[201, 0, 3] = float("nan")
    out = ops.prompt_attention(q, k, v, cu)
    i = torch.arange(290, device=dev)
    seen = i[None] <= i[:, None]
    rest = [d for d in range(D) if d != 3]
    for h in range(2):
        check(out[:201, h], q[:201, h], k[:290, 0], v[:290, 0], seen[:201], D ** -0.5)
        assert not torch.isfinite(out[201:290, h, 3]).any()
        check(out[:290, h][:, rest], q[:290, h], k[:290, 0], v[:290, 0][:, rest], seen, D ** -0.5)


@pytest.mark.parametrize("D", [64, 128])
def test_far_rows(dev, D):
    """The largest stride of tokens, 16 MB, with waves that share rows: tiles of 2 GB."""
    import torch
    from forge_amd import ops
    n, step = 300, 1 << 23
    q, k, v, cu = make([n], 1, 1, D, "float16", dev, 14)
    big = torch.empty(((n - 1) * step + D,), dtype=torch.float16, device=dev)
    far = big.as_strided((n, 1, D), (step, D, 1))
    for causal in (True, False):
        want = ops.prompt_attention(q, k, v, cu, causal=causal)
        far.copy_(k)
        assert torch.equal(ops.prompt_attention(q, far, v, cu, causal=causal), want)
        far.copy_(v)
        assert torch.equal(ops.prompt_attention(q, k, far, cu, causal=causal), want)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,Hq,Hkv", [([300], 1, 1), ([1025, 40], 4, 2), ([2100], 12, 4), ([900], 40, 8), ([130, 7, 61], 3, 3)])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_same_bits_every_call(dev, lens, Hq, Hkv, D, dt):
    """Nothing depends on which wave comes first."""
    import torch
    from forge_amd import ops
    q, k, v, cu = make(lens, Hq, Hkv, D, dt, dev, sum(lens))
    for causal in (True, False):
        want = ops.prompt_attention(q, k, v, cu, causal=causal)
        outs = [ops.prompt_attention(q, k, v, cu, causal=causal) for _ in range(20)]
        for out in outs:
            assert torch.equal(out, want)
