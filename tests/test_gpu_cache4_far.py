"""GPU: cache4_attention where scores and values lie at the ends of what their types hold."""
import pytest

from helpers import say
from test_gpu_cache4 import Cache4, check_all
from test_gpu_cache_attention import drafts_seen, queries, random_tree

pytestmark = pytest.mark.gpu

# (lengths, T, Hq, Hkv, D): one, two, four and eight sets of 16 rows, one chunk and several, by tables and by lengths
CASES = [([300, 40], 1, 4, 1, 64), ([900, 0, 17], 1, 8, 2, 128), ([700], 5, 16, 2, 64), ([500, 31], 61, 4, 1, 128), ([600, 5], 3, 2, 1, 256),
         ([400], 40, 4, 1, 256), ([5000, 3], 1, 8, 2, 128), ([2500, 60], 16, 4, 2, 80)]


def far(c, q, tree, b, h, scale):
    """A head's (result of its best keys, whether they are far enough above the others to be all of it, how far one score may be off):
    in 64 bits, the score's error as in cache4_plain.attention."""
    import torch
    T, D = q.shape[1], q.shape[3]
    group = q.shape[2] // c.cache.shape[1]
    n = c.keys[b][0].shape[0] - T
    k, _, _, step, up, least = (t[:, h // group] for t in c.keys[b])
    v = c.values[b][0][:, h // group]
    x = q[b, :, h].double()
    seen = torch.cat([torch.ones((T, n), dtype=torch.bool), drafts_seen(tree, b, T)], 1).to(q.device)
    s = ((x @ k.T) * scale).masked_fill(~seen, float("-inf"))
    mag = ((x.abs() @ up.abs().T + x.abs().sum(-1, keepdim=True) * least.abs()) * scale).masked_fill(~seen, 0.0).amax(-1)
    groups = x.abs().view(T, D // 8, 8).amax(-1).sum(-1)
    ds = 7 * 2.0 ** -18 * scale * groups * step.max() + (D / 8 + 14) * 2.0 ** -23 * mag
    best, at = s.topk(min(2, s.shape[1]), -1)
    alone = best[:, 0] - best[:, -1] > 4 * ds + 100.0 if s.shape[1] > 1 else torch.ones(T, dtype=torch.bool, device=q.device)
    return v[at[:, 0]], alone, v


@pytest.mark.parametrize("dt,q_size,k_size", [("float16", 2e3, 2e3), ("float16", 2e4, 2e4), ("float16", 6e4, 3e4), ("float16", 6e4, 6e4), ("bfloat16", 1e5, 1e5),
                                              ("bfloat16", 1e10, 1e9), ("bfloat16", 1e16, 1e16), ("bfloat16", 1e3, 1e30)])
@pytest.mark.parametrize("rising", [False, True])
def test_large_scores(dev, dt, q_size, k_size, rising):
    """Scores far from zero, in any order or growing from key to key: a result is the value of its row's best key, where no other's score is
    near, and never outside the values."""
    import torch
    from forge_amd import ops
    d = getattr(torch, dt)
    top = torch.finfo(d).max
    said = 0
    for i, (lens, T, Hq, Hkv, D) in enumerate(CASES):
        say(f"cache4_attention large scores {dt} {q_size} {k_size} rising={rising} lens={lens} T={T} heads={Hq}/{Hkv} D={D}")
        q = queries(len(lens), T, Hq, D, dt, dev, 60 + i)
        sign = torch.where(q[0, 0, 0] < 0, -1.0, 1.0)
        q = (q.float() * q_size).clamp(-top, top).to(d)
        if rising:
            q = (q.float().abs() * sign).to(d)

        def change(b, k, v):
            x = k.float() * (k_size / 1.5)
            if rising:
                x = x.abs() * sign * torch.linspace(0.05, 1.0, x.shape[0], device=dev)[:, None, None]
            k.copy_(x.clamp(-top, top).to(d))
        c = Cache4(lens, T, Hkv, D, 16, dt, dev, 61 + i, change=change)
        tree = random_tree(len(lens), T, 62 + i) if T > 1 else None
        out = ops.cache4_attention(q, c.cache, c.table, c.lens, tree=None if tree is None else tree.to(dev))
        assert torch.isfinite(out).all()
        u = torch.finfo(d).eps / 2
        for b in range(len(lens)):
            for h in range(Hq):
                want, alone, v = far(c, q, tree, b, h, D ** -0.5)
                said += int(alone.sum())
                got = out[b, :, h].double()
                # the best key's weight and value: the weight's 2^-11 of s' 7.5 or less, the products' 2^-18 and the result's own rounding
                room = u * want.abs() + (2.0 ** -11 + 2.0 ** -14) * 9.0 * v.abs().amax() / 7.5 + 2.0 ** -24
                assert ((got - want).abs() <= room)[alone].all(), (b, h)
                assert (got.abs() <= v.abs().amax() * (1 + 2.0 ** -7)).all(), (b, h)
    assert said > 50


@pytest.mark.parametrize("q_size,k_size", [(1e-37, 1e38), (1e-37, 3e38), (3e-30, 1e30), (1e30, 3e-30), (1e35, 1e-35)])
def test_large_and_small(dev, q_size, k_size):
    """BF16 scores of usual size whose factors lie at the ends of the type's range."""
    import torch
    from forge_amd import ops
    top = torch.finfo(torch.bfloat16).max
    for i, (lens, T, Hq, Hkv, D) in enumerate(CASES):
        say(f"cache4_attention large and small {q_size} {k_size} lens={lens} T={T} heads={Hq}/{Hkv} D={D}")
        q = (queries(len(lens), T, Hq, D, "bfloat16", dev, 80 + i).float() * q_size).to(torch.bfloat16)
        c = Cache4(lens, T, Hkv, D, 16, "bfloat16", dev, 81 + i, change=lambda b, k, v: k.copy_((k.float() / 1.5 * k_size).clamp(-top, top).to(k.dtype)))
        tree = random_tree(len(lens), T, 82 + i) if T > 1 else None
        out = ops.cache4_attention(q, c.cache, c.table, c.lens, tree=None if tree is None else tree.to(dev))
        assert torch.isfinite(out).all()
        check_all(out, q, c, lens, tree)


def test_largest_steps(dev):
    """Tiny queries of one sign over BF16 keys that span the type: their products with the integers times a step pass FP32."""
    import torch
    from forge_amd import ops
    top = torch.finfo(torch.bfloat16).max
    for i, (lens, T, Hq, Hkv, D) in enumerate(CASES):
        say(f"cache4_attention largest steps lens={lens} T={T} heads={Hq}/{Hkv} D={D}")
        q = ((1.0 + 0.05 * queries(len(lens), T, Hq, D, "bfloat16", dev, 90 + i).float()) * 1e-38).to(torch.bfloat16)

        def change(b, k, v):
            x = k.float() / 1.5
            x[:, :, 1::7] /= 3.0
            k.copy_((torch.where(x > -1.0, 1.0, -1.0) * top * (1.0 - x.abs().clamp_max(2.0) / 4.0)).to(k.dtype))
        c = Cache4(lens, T, Hkv, D, 16, "bfloat16", dev, 91 + i, change=change)
        tree = random_tree(len(lens), T, 92 + i) if T > 1 else None
        out = ops.cache4_attention(q, c.cache, c.table, c.lens, tree=None if tree is None else tree.to(dev))
        assert torch.isfinite(out).all()
        check_all(out, q, c, lens, tree)


@pytest.mark.parametrize("e", [-60, -100, -108])
def test_equal_small_values(dev, e):
    """Means of BF16 values near the lower end of its range keep their bits."""
    import torch
    from forge_amd import ops
    for i, (lens, T, Hq, Hkv, D) in enumerate(CASES):
        say(f"cache4_attention values of 2^{e} lens={lens} T={T} heads={Hq}/{Hkv} D={D}")
        c = Cache4(lens, T, Hkv, D, 16, "bfloat16", dev, 100 + i, change=lambda b, k, v: v.fill_(2.0 ** e))
        out = ops.cache4_attention(queries(len(lens), T, Hq, D, "bfloat16", dev, 101 + i), c.cache, c.table, c.lens)
        assert (out == 2.0 ** e).all()


@pytest.mark.parametrize("e", [-100, -118, -120, -122])
def test_smallest_steps(dev, e):
    """Steps 2^e of BF16 values over 30001 keys with equal scores: all weights are 2^-26, and 2^(e - 26 + 127), a number of FP16, behind the row's
    factor, so that every product and sum is exact. (With a factor of 2^120 the weights of the last two were zero.)"""
    import torch
    from forge_amd import ops
    n, D = 30000, 64
    say(f"cache4_attention steps of 2^{e}")

    def change(b, k, v):
        k.zero_()
        v.fill_(15.0 * 2.0 ** e)
        v[:, :, 5] = 0.0
        v[:, :, 60] = 3.0 * 2.0 ** e
    c = Cache4([n], 1, 1, D, 16, "bfloat16", dev, 110, change=change)
    out = ops.cache4_attention(queries(1, 1, 3, D, "bfloat16", dev, 111), c.cache, c.table, c.lens)
    want = torch.full((D,), 15.0 * 2.0 ** e, device=dev).to(torch.bfloat16)
    want[5], want[60] = 0.0, 3.0 * 2.0 ** e
    assert torch.equal(out[0, 0], want.expand(3, D))
