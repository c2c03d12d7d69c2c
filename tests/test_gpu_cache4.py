"""GPU: the 4-bit cache: cache4_write and cache4_read bit for bit against the definition, cache4_attention within the bound
of cache4_plain.py."""
import pytest

import cache4_plain as plain
from helpers import say
from test_gpu_cache_attention import drafts_seen, queries, random_tree

pytestmark = pytest.mark.gpu


def heads(T, H, D, dt, dev, seed, spread=1.5):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, H, D), generator=g) * spread
    x[:, :, ::7] *= 3.0
    return x.to(getattr(torch, dt)).to(dev)


def stored(x, D, dt):
    """The 16-bit values that reading back gives."""
    return plain.held(x)[0].float().to(x.dtype)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,Hkv,D,page", [(1, 1, 8, 16), (7, 3, 64, 16), (33, 2, 72, 32), (5, 8, 96, 16), (129, 1, 128, 64), (6, 4, 160, 16),
                                          (18, 2, 192, 128), (40, 5, 256, 16)])
def test_write_read(dev, dt, T, Hkv, D, page):
    import torch
    from forge_amd import ops
    say(f"cache4 write/read {dt} T={T} heads={Hkv} D={D} page={page}")
    d = getattr(torch, dt)
    pages = T // page + 3
    cache = torch.full(ops.cache4_shape(pages, page, Hkv, D), 0xA5, dtype=torch.uint8, device=dev)
    wide = heads(T, 3 * Hkv + 1, D, dt, dev, T + D)                # heads are strided views of a projection's output
    k, v = wide[:, 1:1 + Hkv], wide[:, 1 + Hkv:1 + 2 * Hkv]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(D))[:T].to(torch.int32)
    if T > 4:
        slots[1], slots[3] = -1, pages * page                      # not in the cache
    live = (slots >= 0) & (slots < pages * page)
    assert ops.cache4_write(k, v, cache, slots.to(dev)) is cache
    nk, nv, num = plain.words(cache, page, D)
    at = slots[live].long()
    for x, n, numbers in ((k, nk, num[..., :2]), (v, nv, num[..., 2:])):
        want, step, low = plain.quantize(x[live.to(dev)])
        got = n[at // page, :, at % page]
        assert torch.equal(got[..., :D].double(), want)
        assert (got[..., D:] == 0).all()
        two = numbers[at // page, :, at % page].contiguous().view(d)
        assert torch.equal(two[..., 0].double(), step) and torch.equal(two[..., 1].double(), low)
    # nothing else was touched: no byte of other rows
    other = torch.ones(pages * page, dtype=torch.bool)
    other[at] = False
    rest = torch.arange(pages * page)[other]
    a5 = torch.tensor([0xA5, 0xA5], dtype=torch.uint8).view(torch.int16)
    assert (num[rest // page, :, rest % page] == a5).all()
    for n in (nk, nv):
        assert ((n[rest // page, :, rest % page] == 0xA) | (n[rest // page, :, rest % page] == 0x5)).all()
    rk, rv = ops.cache4_read(cache, slots.to(dev), D, d)
    for x, r in ((k, rk), (v, rv)):
        assert torch.equal(r[live.to(dev)], stored(x[live.to(dev)], D, dt))
        assert (r[~live.to(dev)] == 0).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
def test_write_edges(dev, dt):
    """Heads of one value, of the type's largest and smallest, and with infinities and NaN."""
    import torch
    from forge_amd import ops
    d, D, page = getattr(torch, dt), 64, 16
    info = torch.finfo(d)
    x = torch.randn((8, 2, D), generator=torch.Generator().manual_seed(3)).to(d)
    x[0] = 0.0
    x[1] = -3.5
    x[2, 0, ::2], x[2, 0, 1::2] = info.max, info.min
    x[2, 1] = info.max
    x[3] = x[3] * info.smallest_normal                              # subnormal numbers, steps of zero among them
    x[4, 0, 5] = float("nan")
    x[4, 1, 63] = float("inf")
    x[5, 0, 0] = float("-inf")
    x[6, 0] = info.max
    x[6, 0, 9] = info.max * 0.99
    x = x.to(dev)
    cache = torch.zeros(ops.cache4_shape(2, page, 2, D), dtype=torch.uint8, device=dev)
    slots = torch.arange(4, 12, dtype=torch.int32, device=dev)
    ops.cache4_write(x, x, cache, slots)
    k, v = ops.cache4_read(cache, slots, D, d)
    want = stored(x, D, dt)
    assert torch.equal(k.isnan(), want.isnan()) and torch.equal(v.isnan(), want.isnan())
    assert torch.equal(k.nan_to_num(0.0), want.nan_to_num(0.0)) and torch.equal(v.nan_to_num(0.0), want.nan_to_num(0.0))
    ok = torch.isfinite(x).all(-1)
    assert torch.isfinite(k[ok]).all() and k[~ok].isnan().all()
    # half a step, less the step's own rounding toward zero (an ulp of it fifteen times over), and the result's rounding
    err = (k[ok].double() - x[ok].double()).abs().amax(-1)
    span = (x[ok].double().amax(-1) - x[ok].double().amin(-1))
    room = span / 30 + span * info.eps + x[ok].double().abs().amax(-1) * info.eps / 2 + 16 * info.smallest_normal * info.eps
    assert (err <= room).all()


def test_write_refusals(dev):
    import torch
    from forge_amd import ops
    k = torch.zeros((3, 2, 64), dtype=torch.float16, device=dev)
    cache = torch.zeros(ops.cache4_shape(5, 16, 2, 64), dtype=torch.uint8, device=dev)
    slots = torch.zeros(3, dtype=torch.int32, device=dev)
    for args in ((k, k[:, :1], cache, slots), (k, k, cache[:, :1].contiguous(), slots), (k, k, cache[..., :64].contiguous(), slots),
                 (k, k, cache.view(5, 2, 8, 144), slots), (k, k, cache, slots[:2]), (k.transpose(1, 2), k, cache, slots),
                 (k[..., :60], k[..., :60], cache, slots), (k, k, cache[:0], slots)):
        with pytest.raises(ValueError):
            ops.cache4_write(*args)
    for args in ((k, k.bfloat16(), cache, slots), (k, k, cache.view(torch.int8), slots), (k, k, cache, slots.long()),
                 (k.float(), k.float(), cache, slots)):
        with pytest.raises(TypeError):
            ops.cache4_write(*args)
    with pytest.raises(TypeError):
        ops.cache4_read(cache, slots, 64, torch.float32)
    with pytest.raises(ValueError):
        ops.cache4_read(cache, slots, 128)
    with pytest.raises(ValueError):
        ops.cache4_read(cache, slots[None], 64)
    assert ops.cache4_read(cache, slots[:0], 64)[0].shape == (0, 2, 64)


class Cache4:
    """A 4-bit paged cache whose pages lie in any order; everything that no sequence holds (the ends of last pages,
    pages in between, table entries past the length) is NaN or nonsense."""

    def __init__(self, lens, T, Hkv, D, page, dt, dev, seed, spare=3, width=0, spread=1.5, change=None):
        import torch
        from forge_amd import ops
        g = torch.Generator().manual_seed(seed)
        d = getattr(torch, dt)
        need = [(n + T + page - 1) // page for n in lens]
        pages = sum(need) + spare
        self.cache = torch.full(ops.cache4_shape(pages, page, Hkv, D), 0xFF, dtype=torch.uint8, device=dev)   # NaN in either type
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(max(need), width)), -1, dtype=torch.int32)
        table[:, 1::2] = 1 << 30
        self.keys, self.values, self.rows, at = [], [], [], 0
        for b, n in enumerate(lens):
            ids = order[at:at + need[b]]
            table[b, :need[b]] = ids
            at += need[b]
            k, v = heads(n + T, Hkv, D, dt, dev, seed + 2 * b, spread), heads(n + T, Hkv, D, dt, dev, seed + 2 * b + 1, spread)
            if change:
                change(b, k, v)
            rows = (ids.long()[:, None] * page + torch.arange(page)).flatten()[:n + T].to(torch.int32).to(dev)
            ops.cache4_write(k, v, self.cache, rows)
            self.keys.append(plain.held(k))
            self.values.append(plain.held(v))
            self.rows.append(rows)
        self.table = table.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)


def check_all(out, q, c, lens, tree, scale=None):
    import torch
    B, T, Hq, D = q.shape
    group = Hq // c.cache.shape[1]
    for b, n in enumerate(lens):
        seen = torch.cat([torch.ones((T, n), dtype=torch.bool), drafts_seen(tree, b, T)], 1).to(q.device)
        for h in range(Hq):
            k, v = ([t[:, h // group] for t in x] for x in (c.keys[b], c.values[b]))
            plain.check(out[b, :, h], q[b, :, h], k, v, seen, D ** -0.5 if scale is None else scale)


def run(dev, dt, lens, T, Hq, Hkv, D, page, tree=True, width=0, scale=None, **more):
    from forge_amd import ops
    say(f"cache4_attention {dt} lens={lens} T={T} heads={Hq}/{Hkv} D={D} page={page}")
    c = Cache4(lens, T, Hkv, D, page, dt, dev, 7 * D + T, width=width, **more)
    q = queries(len(lens), T, Hq, D, dt, dev, D + T)
    t = random_tree(len(lens), T, D + T) if tree and T > 1 else None
    out = ops.cache4_attention(q, c.cache, c.table, c.lens, tree=None if t is None else t.to(dev), scale=scale)
    check_all(out, q, c, lens, t, scale)
    return q, c, t, out


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 1, 64), (6, 2, 72), (2, 1, 8), (5, 1, 96), (12, 3, 128), (17, 1, 128), (7, 1, 160), (2, 2, 192),
                                      (16, 2, 256), (1, 1, 80)])
def test_single_tokens(dev, dt, Hq, Hkv, D):
    run(dev, dt, [0, 1, 15, 16, 17, 31, 47, 130, 300], 1, Hq, Hkv, D, 16)


@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_pages(dev, page):
    run(dev, "float16", [63, 64, 65, 500, 1], 1, 8, 2, 128, page)
    run(dev, "bfloat16", [63, 64, 65, 500, 1], 5, 8, 2, 64, page)


@pytest.mark.parametrize("dt,T,Hq,Hkv,D", [("float16", 2, 4, 2, 64), ("bfloat16", 3, 16, 2, 128), ("float16", 7, 21, 3, 96), ("bfloat16", 16, 8, 8, 128),
                                           ("float16", 33, 4, 1, 256), ("bfloat16", 61, 8, 1, 64), ("float16", 64, 16, 2, 192), ("float16", 29, 9, 1, 72),
                                           ("bfloat16", 64, 3, 1, 256), ("float16", 13, 10, 2, 128)])
def test_trees(dev, dt, T, Hq, Hkv, D):
    run(dev, dt, [0, 5, 31, 32, 129, 290], T, Hq, Hkv, D, 16)
    run(dev, dt, [40, 3], T, Hq, Hkv, D, 32, tree=False)


def test_long(dev):
    """Chunks of several workgroups, and their join."""
    run(dev, "float16", [5000, 3, 2047, 2048, 2049], 1, 8, 2, 128, 64)
    run(dev, "bfloat16", [9001, 1], 1, 4, 1, 64, 16)
    run(dev, "float16", [4100], 20, 14, 2, 128, 32)
    run(dev, "bfloat16", [2500, 0], 61, 8, 1, 256, 16)


def test_wide_table(dev):
    """A table much longer than the sequences."""
    run(dev, "float16", [70, 0, 300], 1, 4, 2, 64, 16, width=700)


@pytest.mark.parametrize("dt,T,Hq,Hkv,D,page,lens,width", [
    ("float16", 1, 8, 8, 64, 16, [0, 1, 126, 127, 128, 255, 256, 300, 2000] * 7 + [511, 512], 130),        # more than a wave of sequences
    ("bfloat16", 1, 4, 4, 8, 16, [3] * 64 + [700] + [0] * 70, 130),
    ("float16", 1, 2, 2, 8, 16, [7 * b % 300 for b in range(250)] + [2000, 0, 1000], 700),
    ("float16", 1, 8, 8, 128, 64, [6000, 0, 17], 300),
    ("bfloat16", 1, 4, 1, 256, 32, [0, 9000, 2, 4095], 4100),
    ("bfloat16", 20, 14, 2, 128, 256, [5, 4001], 250),
    ("float16", 64, 8, 1, 256, 256, [0, 2500], 420),
    ("float16", 3, 6, 1, 96, 64, [3000, 1, 129], 2100),
    ("bfloat16", 1, 8, 2, 64, 128, [30000], 1200)])
def test_chunks_by_lengths(dev, dt, T, Hq, Hkv, D, page, lens, width):
    """Tables so long that the chunks' length is made from the sequences' own."""
    from forge_amd import ops
    size = ops.cache4_attention_workspace_size(len(lens), T, Hq, Hkv, D, width * page)
    assert (size - -(-len(lens) // 2) * 16) % (4 * T * Hq * (D + 2)) == 0      # what the first line says holds
    run(dev, dt, lens, T, Hq, Hkv, D, page, width=width)


def test_lengths_between_replays(dev):
    """The lengths change between replays of one graph, and so do the chunks."""
    import torch
    from forge_amd import ops
    full = [6000, 40, 2500]
    c = Cache4(full, 1, 8, 64, 64, "float16", dev, 31, width=300)
    q = queries(3, 1, 8, 64, "float16", dev, 32)
    ws = torch.full((ops.cache4_attention_workspace_size(3, 1, 8, 8, 64, 300 * 64),), 0xFF, dtype=torch.uint8, device=dev)
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.cache4_attention(q, c.cache, c.table, c.lens, workspace=ws, out=out)
    for lens in (full, [0, 0, 0], [6000, 0, 0], [255, 40, 256], [100, 1, 2500], full):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.cache4_attention(q, c.cache, c.table, c.lens))
        for b, n in enumerate(lens):
            for h in range(8):
                k, v = ([t[:n + 1, h] for t in x] for x in (c.keys[b], c.values[b]))
                plain.check(out[b, :, h], q[b, :, h], k, v, torch.ones((1, n + 1), dtype=torch.bool, device=dev), 0.125)


def test_row_that_sees_nothing(dev):
    import torch
    from forge_amd import ops
    c = Cache4([0, 40], 3, 1, 64, 16, "float16", dev, 5)
    q = queries(2, 3, 2, 64, "float16", dev, 6)
    tree = torch.tensor([[0, 2, 0], [0, 2, 7]], dtype=torch.int64, device=dev)
    out = ops.cache4_attention(q, c.cache, c.table, c.lens, tree=tree)
    check_all(out, q, c, [0, 40], tree.cpu())
    assert (out[0, 0] == 0).all() and (out[0, 2] == 0).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
def test_poisoned_drafts(dev, dt):
    """A draft whose key or value holds NaN or infinity reaches the rows that see it, and no bit of the others."""
    import torch
    from forge_amd import ops
    T = 6

    def poison(b, k, v):
        k[-1, 0, 3], v[-2, 0, 5], k[-3, 0, 1] = float("inf"), float("nan"), float("nan")
    clean = Cache4([37, 0], T, 1, 64, 16, dt, dev, 9)
    bad = Cache4([37, 0], T, 1, 64, 16, dt, dev, 9, change=poison)
    q = queries(2, T, 4, 64, dt, dev, 10)
    # tokens 3 to 5 hold the odd ones
    tree = torch.tensor([[1, 2 | 1, 4, 8, 16 | 1, 32 | 2]] * 2, dtype=torch.int64, device=dev)
    a = ops.cache4_attention(q, clean.cache, clean.table, clean.lens, tree=tree)
    b = ops.cache4_attention(q, bad.cache, bad.table, bad.lens, tree=tree)
    assert torch.equal(a[:, :3], b[:, :3]) and torch.isfinite(b[:, :3]).all()
    assert b[:, 3:].isnan().all()


def test_pages_outside_the_cache(dev):
    """Pages that the cache does not have read as zeros: seen, with scores of zero and values of zero."""
    import torch
    from forge_amd import ops
    c = Cache4([64], 1, 1, 64, 16, "float16", dev, 11)
    q = queries(1, 1, 2, 64, "float16", dev, 12)
    c.table[0, 1], c.table[0, 3] = -5, c.cache.shape[0]
    for x in (c.keys[0], c.values[0]):
        for t in x:
            t[16:32] = 0.0
            t[48:64] = 0.0
    out = ops.cache4_attention(q, c.cache, c.table, c.lens)
    check_all(out, q, c, [64], None)
    c.table[:] = 1 << 28
    assert (ops.cache4_attention(q, c.cache, c.table, c.lens) == 0).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
def test_ranges(dev, dt):
    """Scores far from zero, steps of very different sizes, heads of one value, and values as large as the type holds."""
    import torch

    def mixed(b, k, v):
        v[::3] *= 1e-3
        v[1::7] *= 300.0
        v[2::5] = v[2::5, :, :1]                                    # a step of zero
        k[5::9] *= 1e-3
    run(dev, dt, [300, 0, 64], 1, 4, 2, 128, 16, change=mixed)
    run(dev, dt, [150], 9, 4, 2, 64, 16, change=mixed)

    def large(b, k, v):
        v *= (3e3 if dt == "float16" else 1e37)
        k *= 30.0
    _, _, _, out = run(dev, dt, [700, 30], 1, 4, 2, 64, 16, change=large, spread=1.0)
    assert torch.isfinite(out).all()

    def tiny(b, k, v):
        v *= (1e-4 if dt == "float16" else 1e-30)
        k *= 1e-3
    run(dev, dt, [200], 1, 4, 2, 64, 16, change=tiny)
    run(dev, dt, [200], 1, 4, 2, 64, 16, scale=40.0)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("far", [9.0, 13.0, 15.0])
def test_many_small_weights(dev, dt, far):
    """One key far above thousands of others, whose weights are subnormal in FP16 next to its own and still add up."""
    import torch
    from forge_amd import ops
    say(f"cache4_attention small weights {dt} far={far}")
    n, D = 30000, 64
    q = queries(1, 1, 1, D, dt, dev, 40)

    def one(b, k, v):
        k.zero_()
        k[n // 2, 0] = (q[0, 0, 0].float() * (far * 8.0 / q.float().square().sum())).to(k.dtype)
    c = Cache4([n], 1, 1, D, 16, dt, dev, 41, change=one)
    out = ops.cache4_attention(q, c.cache, c.table, c.lens)
    check_all(out, q, c, [n], None)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,D,channel", [(1, 128, 0), (1, 128, 3), (29, 64, 60), (2, 256, 129), (64, 72, 5)])
def test_large_channels(dev, dt, T, D, channel):
    """A channel of queries and keys far above the others, whose products lie next to theirs in the matrix unit."""
    import torch
    from forge_amd import ops
    say(f"large channels {dt} T={T} D={D} channel={channel}")

    def change(b, k, v):
        k[:, :, channel] = 20.0 + k[:, :, channel]
    lens = [700, 0, 33]
    c = Cache4(lens, T, 2, D, 16, dt, dev, 41 + D, change=change, spread=0.5)
    q = queries(3, T, 4, D, dt, dev, 42 + D)
    q[..., channel] = 48.0
    out = ops.cache4_attention(q, c.cache, c.table, c.lens)
    check_all(out, q, c, lens, None)


def test_a_key_between_its_integers(dev):
    """One key with nearly all of the weight, whose values are the middle of its range: the sum of its products, 8 w, is taken off."""
    import torch
    from forge_amd import ops
    D = 64
    k = torch.zeros((16, 1, D), dtype=torch.float16, device=dev)
    v = heads(16, 1, D, "float16", dev, 51, 0.5)
    k[:, 0, 0] = torch.arange(16, device=dev) * -0.5               # weights e^-0.5j
    k[:, 0, 1] = 1.0
    v[0] = 0.0
    v[0, 0, 0], v[0, 0, 1] = -8.0, 7.0                             # step 1, the others 0 = -8 + 8
    cache = torch.zeros(ops.cache4_shape(1, 16, 1, D), dtype=torch.uint8, device=dev)
    ops.cache4_write(k, v, cache, torch.arange(16, dtype=torch.int32, device=dev))
    q = torch.zeros((1, 1, 1, D), dtype=torch.float16, device=dev)
    q[..., 0] = 8.0
    out = ops.cache4_attention(q, cache, torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.full((1,), 15, dtype=torch.int32, device=dev),
                               scale=0.5)
    hk, hv = plain.held(k), plain.held(v)
    plain.check(out[0, 0], q[0, 0], [t[:, 0] for t in hk], [t[:, 0] for t in hv], torch.ones((1, 16), dtype=torch.bool, device=dev), 0.5)


def test_rising_scores(dev):
    """Maxima that grow from tile to tile by far, with steps that fall."""
    def rising(b, k, v):
        import torch
        n = k.shape[0]
        ramp = torch.linspace(0.01, 12.0, n, device=k.device)[:, None, None]
        k.copy_((k.float() * ramp).to(k.dtype))
        v.copy_((v.float() * torch.linspace(3.0, -9.0, n, device=k.device)[:, None, None].exp()).to(v.dtype))
    for dt in ("float16", "bfloat16"):
        run(dev, dt, [1500], 1, 8, 1, 64, 16, change=rising)
        run(dev, dt, [333], 7, 8, 1, 128, 16, change=rising)


def test_queries_that_are_not_finite(dev):
    import torch
    from forge_amd import ops
    c = Cache4([50], 1, 1, 64, 16, "float16", dev, 13)
    q = queries(1, 1, 4, 64, "float16", dev, 14)
    want = ops.cache4_attention(q, c.cache, c.table, c.lens)
    q[0, 0, 1, 5], q[0, 0, 2, 60] = float("nan"), float("-inf")
    q[0, 0, 3] = 0.0
    out = ops.cache4_attention(q, c.cache, c.table, c.lens)
    assert torch.equal(out[0, 0, 0], want[0, 0, 0]) and out[0, 0, 1:3].isnan().all()
    check_all(out[:, :, 3:], q[:, :, 3:], c, [50], None)


@pytest.mark.parametrize("T,dt", [(1, "float16"), (20, "bfloat16")])
def test_same_bits(dev, T, dt):
    """The same call gives the same bits, with a given workspace and without."""
    import torch
    from forge_amd import ops
    lens = [700, 33, 1200]
    q, c, t, out = run(dev, dt, lens, T, 8, 2, 128, 16)
    tree = None if t is None else t.to(dev)
    size = ops.cache4_attention_workspace_size(3, T, 8, 2, 128, c.table.shape[1] * 16)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device=dev)
    buf = torch.empty_like(out)
    for _ in range(20):
        assert ops.cache4_attention(q, c.cache, c.table, c.lens, tree=tree, workspace=ws, out=buf) is buf
        assert torch.equal(buf, out)


def test_attention_refusals(dev):
    import torch
    from forge_amd import ops
    c = Cache4([20], 1, 2, 64, 16, "float16", dev, 15)
    q = queries(1, 1, 4, 64, "float16", dev, 16)
    ok = dict(q=q, cache=c.cache, page_table=c.table, cache_lens=c.lens)
    for bad in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(cache=c.cache[:, :, :, :40].contiguous()), dict(cache=c.cache[0]),
                dict(page_table=c.table[0]), dict(cache_lens=c.lens[None]), dict(tree=torch.zeros((1, 2), dtype=torch.int64, device=dev)),
                dict(scale=0.0), dict(out=q[:, :, :2].contiguous()), dict(q=q.expand(1, 65, 4, 64).contiguous()),
                dict(cache=c.cache.view(c.cache.shape[0] * 2, 2, 8, 72)), dict(cache_lens=c.lens.cpu())):
        with pytest.raises(ValueError):
            ops.cache4_attention(**dict(ok, **bad))
    for bad in (dict(q=q.float()), dict(cache=c.cache.view(torch.int8)), dict(page_table=c.table.long()), dict(tree=c.table)):
        with pytest.raises(TypeError):
            ops.cache4_attention(**dict(ok, **bad))
    long = Cache4([3000], 1, 2, 64, 16, "float16", dev, 17)
    with pytest.raises(ValueError, match="workspace"):
        ops.cache4_attention(q, long.cache, long.table, long.lens, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    assert ops.cache4_attention(q[:0], c.cache, c.table[:0], c.lens[:0]).shape == (0, 1, 4, 64)


def test_other_stream_and_graph(dev):
    """On another stream, and captured twice with one workspace and replayed between eager calls."""
    import torch
    from forge_amd import ops
    lens = [900, 20]
    q, c, _, out = run(dev, "float16", lens, 1, 8, 2, 128, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    size = ops.cache4_attention_workspace_size(2, 1, 8, 2, 128, c.table.shape[1] * 16)
    with torch.cuda.stream(side):
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        got = ops.cache4_attention(q, c.cache, c.table, c.lens, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, out)
    k, v = heads(2, 2, 128, "float16", dev, 21), heads(2, 2, 128, "float16", dev, 22)
    rows = torch.stack([r[-1] for r in c.rows])
    results, graphs = [], []
    for _ in range(2):
        res = torch.empty_like(out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.cache4_write(k, v, c.cache, rows)
            ops.cache4_attention(q, c.cache, c.table, c.lens, workspace=ws, out=res)
        results.append(res)
        graphs.append(g)
    for i in range(4):
        k.copy_(heads(2, 2, 128, "float16", dev, 30 + i))
        for g, res in zip(graphs, results):
            res.zero_()
            g.replay()
            torch.cuda.synchronize()
            eager = ops.cache4_attention(q, c.cache, c.table, c.lens)
            assert torch.equal(res, eager)
    assert not torch.equal(results[0], out)


def test_many_sequences(dev):
    """More sequences than a grid has rows."""
    import torch
    from forge_amd import ops
    B = 66000
    c = Cache4([5, 20, 0], 1, 1, 8, 16, "float16", dev, 23)
    pick = torch.arange(B) % 3
    q = queries(3, 1, 1, 8, "float16", dev, 24)
    small = ops.cache4_attention(q, c.cache, c.table, c.lens)
    out = ops.cache4_attention(q[pick.to(dev)].contiguous(), c.cache, c.table[pick.to(dev)].contiguous(), c.lens[pick.to(dev)].contiguous())
    assert torch.equal(out, small[pick.to(dev)])
    check_all(small, q, c, [5, 20, 0], None)
