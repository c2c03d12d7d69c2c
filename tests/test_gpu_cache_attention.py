"""GPU: cache_attention against the plain 64-bit form, within the bound of attention_plain.py."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu


class Cache:
    """A paged cache of random rows whose pages lie in any order; everything that no sequence holds (the ends of
    last pages, pages in between, table entries past the length) is NaN or nonsense."""

    def __init__(self, lens, T, Hkv, D, page, dt, dev, seed, spare=3, width=0):
        import torch
        g = torch.Generator().manual_seed(seed)
        d = getattr(torch, dt)
        need = [(n + T + page - 1) // page for n in lens]
        pages = sum(need) + spare
        self.k = torch.full((pages, page, Hkv, D), float("nan"), dtype=d, device=dev)
        self.v = torch.full((pages, page, Hkv, D), float("nan"), dtype=d, device=dev)
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(max(need), width)), -1, dtype=torch.int32)
        table[:, 1::2] = 1 << 30
        self.keys, self.values, at = [], [], 0
        for b, n in enumerate(lens):
            ids = order[at:at + need[b]]
            table[b, :need[b]] = ids
            at += need[b]
            k, v = ((torch.randn((n + T, Hkv, D), generator=g) * 1.5).to(d).to(dev) for _ in range(2))
            rows = (ids.long()[:, None] * page + torch.arange(page)).flatten()[:n + T].to(dev)
            self.k.view(-1, Hkv, D)[rows] = k
            self.v.view(-1, Hkv, D)[rows] = v
            self.keys.append(k)
            self.values.append(v)
        self.table = table.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)


def random_tree(B, T, seed):
    """Random trees as bit masks, with a token that sees no draft and one that sees itself only."""
    import random
    import torch
    rng = random.Random(seed)
    rows = []
    for _ in range(B):
        bits = []
        for t in range(T):
            parent = rng.randrange(-1, t) if t else -1
            bits.append((1 << t) | (bits[parent] if parent >= 0 else 0))
        if T > 2:
            bits[T // 2] = 0
        rows.append([m - (1 << 64) if m >> 63 else m for m in bits])
    return torch.tensor(rows, dtype=torch.int64)


def drafts_seen(tree, b, T):
    import torch
    if tree is None:
        return torch.ones((T, T), dtype=torch.bool).tril()
    return torch.tensor([[(int(m) >> j) & 1 == 1 for j in range(T)] for m in tree[b].tolist()])


def check_all(out, q, c, lens, tree, scale=None):
    import torch
    from attention_plain import check
    B, T, Hq, D = q.shape
    group = Hq // c.k.shape[2]
    for b, n in enumerate(lens):
        seen = torch.cat([torch.ones((T, n), dtype=torch.bool), drafts_seen(tree, b, T)], 1).to(q.device)
        for h in range(Hq):
            check(out[b, :, h], q[b, :, h], c.keys[b][:, h // group], c.values[b][:, h // group], seen,
                  D ** -0.5 if scale is None else scale)


def queries(B, T, Hq, D, dt, dev, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, T, Hq, D), generator=g) * 1.5).to(getattr(torch, dt)).to(dev)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,T,Hq,Hkv,D,page", [
    ([0], 1, 1, 1, 8, 1), ([1, 0, 31, 32, 33], 1, 4, 2, 64, 16), ([127, 128, 129, 500], 1, 8, 1, 128, 16),
    ([100], 1, 7, 1, 80, 32), ([1000, 3], 1, 6, 6, 256, 64), ([2500], 1, 2, 2, 96, 4), ([5, 0, 60], 3, 4, 2, 64, 8),
    ([130, 17], 16, 8, 2, 128, 64), ([700], 5, 9, 3, 200, 128), ([300, 0, 64], 64, 2, 1, 64, 16),
    ([200, 31], 61, 8, 1, 128, 32), ([40], 33, 4, 1, 256, 16), ([2049, 4100], 2, 2, 1, 128, 256)])
def test_cache_attention(dev, lens, T, Hq, Hkv, D, page, dt):
    from forge_amd import ops
    c = Cache(lens, T, Hkv, D, page, dt, dev, sum(lens) + T + D)
    q = queries(len(lens), T, Hq, D, dt, dev, T)
    say(f"cache_attention {dt} lens={lens} T={T} Hq={Hq} Hkv={Hkv} D={D} page={page}")
    check_all(ops.cache_attention(q, c.k, c.v, c.table, c.lens), q, c, lens, None)
    tree = random_tree(len(lens), T, T)
    check_all(ops.cache_attention(q, c.k, c.v, c.table, c.lens, tree=tree.to(dev), scale=0.2), q, c, lens, tree, 0.2)


@pytest.mark.parametrize("lens,T,Hq,Hkv,D,page", [
    ([900, 5], 10, 4, 1, 96, 16), ([300], 20, 4, 1, 96, 32), ([600, 0], 10, 4, 1, 64, 16), ([500], 10, 8, 2, 256, 16),
    ([3000, 40], 33, 8, 2, 128, 64), ([5000], 64, 8, 1, 72, 16)])
def test_row_sets(dev, lens, T, Hq, Hkv, D, page):
    """Two and four sets of 32 rows at each head size, and rows enough to lengthen the chunks."""
    from forge_amd import ops
    c = Cache(lens, T, Hkv, D, page, "bfloat16", dev, T + D)
    q = queries(len(lens), T, Hq, D, "bfloat16", dev, D)
    say(f"cache_attention lens={lens} T={T} Hq={Hq} Hkv={Hkv} D={D} page={page}")
    tree = random_tree(len(lens), T, D)
    check_all(ops.cache_attention(q, c.k, c.v, c.table, c.lens, tree=tree.to(dev)), q, c, lens, tree)


def test_table_wider_than_the_lengths(dev):
    """A table laid out for a far longer sequence: many chunks without keys."""
    from forge_amd import ops
    lens = [700, 0, 12]
    c = Cache(lens, 2, 2, 64, 16, "float16", dev, 5, width=1500)
    q = queries(3, 2, 8, 64, "float16", dev, 5)
    check_all(ops.cache_attention(q, c.k, c.v, c.table, c.lens), q, c, lens, None)


def test_rows_that_see_nothing(dev):
    import torch
    from forge_amd import ops
    c = Cache([0, 40], 4, 1, 64, 16, "bfloat16", dev, 6)
    q = queries(2, 4, 2, 64, "bfloat16", dev, 6)
    tree = torch.tensor([[0, 2, 0, 15], [0, 0, 4, 8]], dtype=torch.int64)
    out = torch.full_like(q, 3.0)
    ops.cache_attention(q, c.k, c.v, c.table, c.lens, tree=tree.to(dev), out=out)
    assert (out[0, [0, 2]] == 0).all()
    check_all(out, q, c, [0, 40], tree)


@pytest.mark.parametrize("T,Hq,D", [(6, 2, 128), (40, 4, 64), (5, 1, 256)])
@pytest.mark.parametrize("n", [20, 1000])
def test_masked_drafts_hold_anything(dev, T, Hq, D, n):
    """A drafted token's infinite or NaN key and value reach only the tokens that see it."""
    import torch
    from attention_plain import check
    from forge_amd import ops
    c = Cache([n], T, 1, D, 16, "float16", dev, 7)
    q = queries(1, T, Hq, D, "float16", dev, 7)
    slot = [int(c.table[0, (n + j) // 16]) * 16 + (n + j) % 16 for j in (1, 2)]
    c.v.view(-1, 1, D)[slot[0], 0, 5] = float("inf")
    c.k.view(-1, 1, D)[slot[1]] = float("nan")
    c.v.view(-1, 1, D)[slot[1]] = float("nan")
    tree = torch.tensor([[1 << t for t in range(T)]], dtype=torch.int64)       # every draft on its own
    tree[0, 3] |= 1 << 1
    out = ops.cache_attention(q, c.k, c.v, c.table, c.lens, tree=tree.to(dev))
    rows = [t for t in range(T) if t not in (1, 2, 3)]
    seen = torch.cat([torch.ones((T, n), dtype=torch.bool), drafts_seen(tree, 0, T)], 1).to(dev)
    for h in range(Hq):
        check(out[0, rows, h], q[0, rows, h], c.keys[0][:, 0], c.values[0][:, 0], seen[rows], D ** -0.5)
    assert torch.isnan(out[0, 2]).all()
    assert (out[0, [1, 3], :, 5] == float("inf")).all()
    others = [d for d in range(D) if d != 5]
    assert torch.isfinite(out[0, [1, 3]][..., others]).all()


def test_table_ends_before_the_drafts(dev):
    """Positions past the table are not seen, pages that the cache does not have read as zeros."""
    import torch
    from attention_plain import check
    from forge_amd import ops
    c = Cache([60], 8, 1, 64, 16, "float16", dev, 8)
    q = queries(1, 8, 1, 64, "float16", dev, 8)
    table = c.table[:, :4].contiguous()                                        # 64 positions: drafts 0 to 3
    out = ops.cache_attention(q, c.k, c.v, table, c.lens)
    seen = torch.ones((8, 68), dtype=torch.bool, device=dev).tril(60)
    seen[:, 64:] = False
    check(out[0, :, 0], q[0, :, 0], c.keys[0][:, 0], c.values[0][:, 0], seen, 0.125)
    table = c.table.clone()
    table[0, 1] = c.k.shape[0]
    table[0, 2] = -5
    out = ops.cache_attention(q, c.k, c.v, table, c.lens)
    k, v = c.keys[0][:, 0].clone(), c.values[0][:, 0].clone()
    k[16:48], v[16:48] = 0.0, 0.0
    seen = torch.ones((8, 68), dtype=torch.bool, device=dev).tril(60)
    check(out[0, :, 0], q[0, :, 0], k, v, seen, 0.125)
    lens = torch.tensor([-3], dtype=torch.int32, device=dev)                   # a negative length counts as none
    zero = torch.zeros((1,), dtype=torch.int32, device=dev)
    assert torch.equal(ops.cache_attention(q, c.k, c.v, c.table, lens), ops.cache_attention(q, c.k, c.v, c.table, zero))


def test_cache_past_32_bits(dev):
    """A cache of more than 2^32 elements, read at its end."""
    import torch
    from forge_amd import ops
    page, Hkv, D = 256, 8, 128
    pages = (1 << 32) // (page * Hkv * D) + 8
    k = torch.empty((pages, page, Hkv, D), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    small = Cache([1000], 1, Hkv, D, page, "float16", dev, 9, spare=0)
    n = small.k.shape[0]
    k[-n:], v[-n:] = small.k, small.v
    q = queries(1, 1, 16, D, "float16", dev, 9)
    # entries of the table past the length stay nonsense
    table = torch.where((small.table >= 0) & (small.table < n), small.table + (pages - n), small.table)
    assert torch.equal(ops.cache_attention(q, k, v, table, small.lens),
                       ops.cache_attention(q, small.k, small.v, small.table, small.lens))


def test_same_bits_alone_and_in_a_batch(dev):
    """A sequence's result does not change from call to call, nor with dirty workspaces."""
    import torch
    from forge_amd import ops
    lens = [900, 33, 2000]
    c = Cache(lens, 4, 2, 128, 16, "float16", dev, 10)
    q = queries(3, 4, 8, 128, "float16", dev, 10)
    size = ops.cache_attention_workspace_size(3, 4, 8, 2, 128, c.table.shape[1] * 16)
    assert size > 0
    ws = torch.full((size,), 255, dtype=torch.uint8, device=dev)
    want = ops.cache_attention(q, c.k, c.v, c.table, c.lens)
    for _ in range(3):
        assert torch.equal(ops.cache_attention(q, c.k, c.v, c.table, c.lens, workspace=ws), want)


def test_graph_and_stream(dev):
    import torch
    from forge_amd import ops
    lens = [300, 90]
    c = Cache(lens, 8, 2, 64, 16, "float16", dev, 11)
    q = queries(2, 8, 4, 64, "float16", dev, 11)
    size = ops.cache_attention_workspace_size(2, 8, 4, 2, 64, c.table.shape[1] * 16)
    ws = torch.empty((max(size, 16),), dtype=torch.uint8, device=dev)
    out = torch.empty_like(q)
    want = ops.cache_attention(q, c.k, c.v, c.table, c.lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_attention(q, c.k, c.v, c.table, c.lens, out=out, workspace=ws)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_attention(q, c.k, c.v, c.table, c.lens, out=out, workspace=ws)
    for _ in range(3):
        q.mul_(0.5)
        c.lens.sub_(7)                                               # lengths are read on the device
        want = ops.cache_attention(q, c.k, c.v, c.table, c.lens)
        out.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(dev):
    import torch
    from forge_amd import ops
    c = Cache([30], 2, 2, 64, 16, "float16", dev, 12)
    q = queries(1, 2, 4, 64, "float16", dev, 12)
    f = ops.cache_attention
    tree = torch.zeros((1, 2), dtype=torch.int64, device=dev)
    for bad in (lambda: f(q.float(), c.k, c.v, c.table, c.lens), lambda: f(q, c.k.to(torch.bfloat16), c.v, c.table, c.lens),
                lambda: f(q, c.k, c.v, c.table.long(), c.lens), lambda: f(q, c.k, c.v, c.table, c.lens.long()),
                lambda: f(q, c.k, c.v, c.table, c.lens, tree=tree.int())):
        with pytest.raises(TypeError):
            bad()
    many = torch.zeros((1, 65, 4, 64), dtype=torch.float16, device=dev)
    for bad in (lambda: f(q[0], c.k, c.v, c.table, c.lens), lambda: f(many, c.k, c.v, c.table, c.lens),
                lambda: f(many[:, :0], c.k, c.v, c.table, c.lens), lambda: f(q[:, :, :3].contiguous(), c.k, c.v, c.table, c.lens),
                lambda: f(q.transpose(1, 2), c.k, c.v, c.table, c.lens), lambda: f(q, c.k, c.v[:1], c.table, c.lens),
                lambda: f(q, c.k[:, :12].contiguous(), c.v[:, :12].contiguous(), c.table, c.lens),
                lambda: f(q, c.k[:, ::2], c.v[:, ::2], c.table, c.lens), lambda: f(q, c.k, c.v, c.table[0], c.lens),
                lambda: f(q, c.k, c.v, c.table, c.lens.repeat(2)), lambda: f(q, c.k, c.v, c.table, c.lens, tree=tree[:, :1]),
                lambda: f(q, c.k, c.v, c.table, c.lens, scale=0.0), lambda: f(q, c.k.cpu(), c.v, c.table, c.lens),
                lambda: f(q, c.k, c.v, c.table, c.lens, out=torch.empty((1, 2, 4, 32), dtype=q.dtype, device=dev))):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros((1, 100), dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        f(q, c.k, c.v, wide, c.lens, workspace=torch.empty((16,), dtype=torch.uint8, device=dev))


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,T,Hq,Hkv", [([1000], 1, 4, 1), ([700, 3, 1500], 5, 16, 2), ([900, 2000], 12, 16, 4),
                                           ([1200, 40], 61, 8, 2), ([3000] * 8, 1, 32, 8)])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_same_bits_every_call(dev, lens, T, Hq, Hkv, D, dt):
    """Nothing depends on which wave or workgroup comes first."""
    import torch
    from forge_amd import ops
    c = Cache(lens, T, Hkv, D, 16, dt, dev, D)
    q = queries(len(lens), T, Hq, D, dt, dev, D)
    want = ops.cache_attention(q, c.k, c.v, c.table, c.lens)
    outs = [ops.cache_attention(q, c.k, c.v, c.table, c.lens) for _ in range(20)]
    for out in outs:
        assert torch.equal(out, want)
