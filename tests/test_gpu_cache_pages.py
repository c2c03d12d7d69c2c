"""GPU: fork_pages against the same rules row by row on the host, exactly, and copy_pages against indexing."""
import random

import pytest

from helpers import say

pytestmark = pytest.mark.gpu


def plain_fork(table, lens, parents, refs, page):
    """The documented rules, row by row, on lists."""
    rows, width, pages = len(table), len(table[0]), len(refs)
    group = len(parents[0])
    ok = lambda p: 0 <= p < pages                                   # noqa: E731
    counts = list(refs)
    for row in table:
        for p in row:
            if ok(p):
                counts[p] -= 1
    free = [p for p in range(pages) if refs[p] == 0]
    out = dict(table=[], lens=[], slots=[], src=[], dst=[])
    children = set()
    for r in range(rows):
        up = parents[r // group][r % group]
        row, slot, a, b, n = [-1] * width, -1, -1, -1, 0
        if 0 <= up < group:
            up += r // group * group
            n = min(max(lens[up], 0), width * page)
            at = n // page
            row[:at] = [p if ok(p) else -1 for p in table[up][:at]]
            if at < width:
                last = table[up][at] if ok(table[up][at]) else -1
                if up not in children and last >= 0 and refs[last] == 1:
                    mine = last
                else:
                    mine = free.pop(0) if free else -1
                    if mine >= 0 and last >= 0 and n % page:
                        a, b = last, mine
                row[at] = mine
                slot = mine * page + n % page if mine >= 0 else -1
            children.add(up)
        for p in row:
            if p >= 0:
                counts[p] += 1
        for key, x in (("table", row), ("lens", n), ("slots", slot), ("src", a), ("dst", b)):
            out[key].append(x)
    out["refs"] = counts
    return out


def state(requests, group, width, page, pages, seed, most=None, shared=True):
    """Rows of random lengths that share the full pages of a beginning, as searches leave them, with the counts."""
    rng = random.Random(seed)
    order = list(range(pages))
    rng.shuffle(order)
    table, lens = [], []
    for _ in range(requests):
        n = rng.randint(0, (most or width * page) - 1)
        same = [order.pop() for _ in range(rng.randint(0, n // page))] if shared else []
        for _ in range(group):
            own = (n + page - 1) // page - len(same)
            row = same + [order.pop() for _ in range(own)]
            table.append(row + [-1] * (width - len(row)))
            lens.append(n)
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    parents = [[rng.choice([-1, rng.randrange(group), rng.randrange(group), min(1, group - 1)]) for _ in range(group)] for _ in range(requests)]
    return table, lens, parents, refs


def on(dev, *lists):
    import torch
    return [torch.tensor(x, dtype=torch.int32, device=dev) for x in lists]


def check(dev, table, lens, parents, refs, page, **more):
    from forge_amd import ops
    got = ops.fork_pages(*on(dev, table, lens, parents, refs), page, **more)
    want = plain_fork(table, lens, parents, refs, page)
    for key in want:
        assert getattr(got, key).cpu().tolist() == want[key], key
    return got, want


@pytest.mark.parametrize("requests,group,width,page,pages", [(1, 1, 1, 1, 3), (1, 4, 5, 16, 40), (3, 5, 30, 4, 700), (64, 8, 9, 16, 6000), (2, 300, 3, 8, 2500),
                                                            (1000, 8, 2, 32, 20000), (7, 3, 260, 2, 9001), (8192, 1, 1, 16, 9000), (512, 2, 4, 256, 2048), (513, 2, 4, 256, 2048),
                                                            (8, 4, 128, 1, 2048), (8, 4, 128, 1, 2049)])
def test_sizes(dev, requests, group, width, page, pages):
    for seed in range(3):
        say(f"fork_pages {requests} x {group} width={width} page={page} pages={pages} seed={seed}")
        table, lens, parents, refs = state(requests, group, width, page, pages, seed, most=min(width * page, 200))
        got, want = check(dev, table, lens, parents, refs, page)
        # the counts are the names again, and copied pages are nobody else's
        counts = [0] * pages
        for row in want["table"]:
            for p in row:
                if p >= 0:
                    counts[p] += 1
        assert counts == want["refs"]
        fresh = [d for d in want["dst"] if d >= 0]
        assert len(set(fresh)) == len(fresh) and not set(fresh) & set(want["src"]) - {-1}


def test_chain(dev):
    """Twenty steps of searches, each on the last one's table, while the pages run through the pool."""
    import torch
    from forge_amd import ops
    R, G, P, pages, width = 6, 4, 4, 200, 12
    rng = random.Random(5)
    table, lens, parents, refs = state(R, G, width, P, pages, 5, most=10)
    t = on(dev, table, lens, parents, refs)
    for step in range(20):
        want = plain_fork(table, lens, parents, refs, P)
        got = ops.fork_pages(*t, P)
        for key in want:
            assert getattr(got, key).cpu().tolist() == want[key], (step, key)
        table, refs = want["table"], want["refs"]
        lens = [n + (s >= 0) for n, s in zip(want["lens"], want["slots"])]
        parents = [[rng.randrange(G) for _ in range(G)] for _ in range(R)]
        t = [got.table, got.lens + (got.slots >= 0).to(torch.int32), *on(dev, parents), got.refs]


def test_no_room(dev):
    """No free page, fewer than rows that need one, and rows whose table is full."""
    table, lens = [[0, 1, -1], [2, -1, -1], [3, 4, 5], [6, 7, 8]], [8, 2, 12, 11]
    refs = [1] * 9
    for parents in ([[0, 0, 2, 3]], [[1, 1, 1, 1]], [[3, 3, 3, 3]], [[2, 2, -1, 7]]):
        check(dev, table, lens, parents, refs, 4)
        check(dev, table, lens, parents, refs + [0], 4)
        check(dev, table, lens, parents, [0] * 0 + refs + [0, 5, 0], 4)


def test_shared_last_page(dev):
    """A page in use that others name (another table, or two rows of this one) is copied even for its first child."""
    check(dev, [[0, 1], [0, 2]], [6, 6], [[0, 1]], [2, 2, 1, 0, 0], 4)
    check(dev, [[0, 1], [0, 1]], [6, 6], [[0, 1]], [2, 2, 0, 0, 0], 4)
    check(dev, [[0, 1], [0, 1]], [6, 6], [[1, 1]], [2, 2, 0, 0, 0], 4)


def test_odd_inputs(dev):
    """Table entries, parents and lengths that are none."""
    big = (1 << 31) - 1
    check(dev, [[0, -7, 99], [1, big, 2], [3, 4, 5]], [9, 5, big], [[0, 1, 2]], [1] * 6 + [0] * 4, 4)
    check(dev, [[0, 1, 2], [3, 4, 5]], [-5, 3], [[0, 0]], [1] * 6 + [0] * 4, 4)
    check(dev, [[0, 1, 2], [3, 4, 5]], [7, 3], [[-big - 1, 2]], [1] * 6 + [0] * 4, 4)
    check(dev, [[0, 1, 2], [3, 4, 5]], [0, 0], [[0, 1]], [1] * 6 + [0] * 4, 4)       # a page taken ahead is kept


def test_far_free_page(dev):
    """The free pages lie at the end of a large pool, in its last, ragged part."""
    import torch
    from forge_amd import ops
    pages = 300000
    refs = torch.ones(pages, dtype=torch.int32, device=dev)
    refs[-3:] = 0
    refs[123456] = 0
    table = torch.tensor([[5], [6], [7], [8], [9]], dtype=torch.int32, device=dev)
    got = ops.fork_pages(table, *on(dev, [3] * 5, [[0, 0, 0, 0, 0]]), refs, 16)
    assert got.slots.tolist() == [5 * 16 + 3, 123456 * 16 + 3, (pages - 3) * 16 + 3, (pages - 2) * 16 + 3, (pages - 1) * 16 + 3]
    want = refs.clone()
    want[[6, 7, 8, 9]] -= 1
    want[[123456, -3, -2, -1]] += 1
    assert torch.equal(got.refs, want)


def test_buffers_graph_and_stream(dev):
    import torch
    from forge_amd import ops
    table, lens, parents, refs = state(5, 4, 9, 16, 400, 3)
    t = on(dev, table, lens, parents, refs)
    want = ops.fork_pages(*t, 16)
    ws = torch.full((ops.fork_pages_workspace_size(20, 400),), 0xFF, dtype=torch.uint8, device=dev)
    out = ops.Forked(*(torch.full_like(x, 77) for x in want))
    assert ops.fork_pages(*t, 16, workspace=ws, out=out) is out
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.fork_pages(*t, 16)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    cache = torch.randn((400, 16, 8), device=dev)
    keep = cache.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.fork_pages(*t, 16, workspace=ws, out=out)
        ops.copy_pages([cache], out.src, out.dst)
    for seed in range(4):
        table, lens, parents, refs = state(5, 4, 9, 16, 400, seed)
        for x, y in zip(t, on(dev, table, lens, parents, refs)):
            x.copy_(y)
        cache.copy_(keep)
        g.replay()
        torch.cuda.synchronize()
        eager = ops.fork_pages(*t, 16)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        wanted = keep.clone()
        on_ = eager.dst >= 0
        wanted[eager.dst[on_].long()] = keep[eager.src[on_].long()]
        assert torch.equal(cache, wanted)


@pytest.mark.parametrize("shape,dt,tensors", [((9, 4), "float32", 1), ((40, 16, 2, 64), "float16", 3), ((70, 16, 1, 72), "uint8", 2), ((7, 8), "int64", 70),
                                              ((33, 5, 1000, 2), "float32", 4), ((3, 1, 16), "uint8", 260)])
def test_copy(dev, shape, dt, tensors):
    import torch
    from forge_amd import ops
    say(f"copy_pages {shape} {dt} x {tensors}")
    g = torch.Generator(device=dev).manual_seed(1)
    caches = [torch.randint(0, 200, shape, generator=g, device=dev).to(getattr(torch, dt)) for _ in range(tensors)]
    pages = shape[0]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).tolist()
    half = pages // 2
    src, dst = order[:half], order[half:2 * half]
    src += [-1, 0, pages, src[0]]                                    # none of these is a pair; the last one is, twice from one page
    dst += [0, -1, 0, order[-1] if pages % 2 else -1]
    want = [t.clone() for t in caches]
    for t in want:
        for a, b in zip(src, dst):
            if 0 <= a < pages and 0 <= b < pages:
                t[b] = t[a]
    ops.copy_pages(caches if tensors % 2 else tuple(caches), *on(dev, src, dst))
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_copy_many_pairs(dev):
    """More pairs than a grid has rows."""
    import torch
    from forge_amd import ops
    cache = torch.arange(150000, dtype=torch.int32, device=dev)[:, None].repeat(1, 4).contiguous()
    n = 70000
    src = torch.arange(n, dtype=torch.int32, device=dev)
    ops.copy_pages([cache], src, src + n)
    assert torch.equal(cache[n:2 * n], cache[:n]) and cache[2 * n, 0] == 2 * n


def test_copy_past_2_gb(dev):
    """Pages whose offsets pass 32 bits."""
    import torch
    from forge_amd import ops
    cache = torch.zeros((70000, 1 << 16), dtype=torch.uint8, device=dev)
    cache[2] = 7
    cache[69999, ::3] = 5
    keep = cache[69999].clone()
    ops.copy_pages([cache], *on(dev, [2, 69999], [69998, 1]))
    assert (cache[69998] == 7).all() and torch.equal(cache[1], keep) and cache[0].sum() == 0


def test_refusals(dev):
    import torch
    from forge_amd import ops
    t = on(dev, [[0, 1], [2, -1]], [5, 2], [[0, 1]], [1, 1, 1, 0])
    for i, bad in ((0, t[0][0]), (1, t[1][None]), (1, t[1][:1]), (2, t[2][0]), (2, t[2][:, :1].contiguous()), (3, t[3][None]), (3, t[3][:0])):
        with pytest.raises(ValueError):
            ops.fork_pages(*(bad if i == j else x for j, x in enumerate(t)), 4)
    for page in (0, 3, -4, 4.0, True, 1 << 30):
        with pytest.raises(ValueError):
            ops.fork_pages(*t, page)
    with pytest.raises(TypeError):
        ops.fork_pages(t[0].long(), *t[1:], 4)
    with pytest.raises(ValueError):
        ops.fork_pages(t[0].cpu(), *t[1:], 4)
    out = ops.fork_pages(*t, 4)
    from forge_amd import _lib
    ws = torch.empty(ops.fork_pages_workspace_size(2, 4), dtype=torch.uint8, device=dev)
    for same in (out._replace(table=t[0]), out._replace(refs=t[3])):
        with pytest.raises(_lib.ForgeError):
            ops.fork_pages(*t, 4, workspace=ws, out=same)
    with pytest.raises(ValueError):
        ops.fork_pages(*t, 4, workspace=ws[:4], out=out)
    with pytest.raises(ValueError):
        ops.fork_pages(*t, 4, workspace=ws, out=out._replace(slots=out.slots[:1]))
    c = torch.zeros((4, 16), device=dev)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    for caches in ([c, c[:3]], [c, c.half()], [c.t()], [c[:0]], [torch.zeros((4, 3), device=dev)], [c.cpu()]):
        with pytest.raises(ValueError):
            ops.copy_pages(caches, i, i)
    with pytest.raises(TypeError):
        ops.copy_pages([c, None], i, i)
    with pytest.raises(TypeError):
        ops.copy_pages([c], i.long(), i)
    with pytest.raises(ValueError):
        ops.copy_pages([c], i, torch.zeros(2, dtype=torch.int32, device=dev))
    ops.copy_pages([], i, i)
    ops.copy_pages([c], i[:0], i[:0])
