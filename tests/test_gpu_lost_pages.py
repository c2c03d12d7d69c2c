"""GPU: pools of pages that run out. A row that found no page to copy its last tokens into ends with the next call, however many
pages are free then; every other row's pages hold its own tokens. A search's rows whose newest token found no slot have no continuation."""
import random

import pytest

from helpers import say
from test_gpu_beam_select import check as check_selection
from test_gpu_cache4 import stored
from test_gpu_cache_pages import on, plain_fork, state

pytestmark = pytest.mark.gpu

KEYS = ("table", "lens", "slots", "src", "dst", "refs")


def lost(row, n, page):
    """Whether a row has tokens on a page that it does not name."""
    at = min(n, len(row) * page) // page
    return n > 0 and at < len(row) and n % page != 0 and row[at] < 0


def plain(table, lens, parents, refs, page):
    """plain_fork, rows that go on from a lost one ending."""
    group = len(parents[0])
    gone = [lost(row, n, page) for row, n in zip(table, lens)]
    left = [[-1 if 0 <= p < group and gone[b * group + p] else p for p in row] for b, row in enumerate(parents)]
    return plain_fork(table, lens, left, refs, page)


def test_two_calls(dev):
    """Two rows over a full pool: the second finds no page for its copy, and is no row of the next call, in which a page is free."""
    from forge_amd import ops
    table, lens, refs = [[0, 1], [2, 3]], [6, 6], [1] * 8
    t = on(dev, table, lens, [[0, 0]], refs)
    a = ops.fork_pages(*t, 4)
    assert a.table.tolist() == [[0, 1], [0, -1]] and a.lens.tolist() == [6, 6] and a.slots.tolist() == [6, -1]
    assert a.refs.tolist() == [2, 1, 0, 0, 1, 1, 1, 1] and a.dst.tolist() == [-1, -1]
    b = ops.fork_pages(a.table, a.lens, *on(dev, [[0, 1]]), a.refs, 4)
    assert b.table.tolist() == [[0, 1], [-1, -1]] and b.lens.tolist() == [6, 0] and b.slots.tolist() == [6, -1]
    assert b.refs.tolist() == [1, 1, 0, 0, 1, 1, 1, 1] and b.src.tolist() == b.dst.tolist() == [-1, -1]


@pytest.mark.parametrize("requests,group,width,page,pages", [(1, 4, 5, 16, 40), (8, 4, 9, 4, 700), (300, 4, 3, 8, 2048), (300, 4, 9, 8, 9000), (2, 300, 9, 8, 6000)])
def test_rows_without_their_last_page(dev, requests, group, width, page, pages):
    from forge_amd import ops
    for seed in range(4):
        say(f"fork_pages, rows without a page, {requests} x {group} width={width} page={page} pages={pages} seed={seed}")
        table, lens, parents, refs = state(requests, group, width, page, pages, seed)
        rng = random.Random(seed)
        for r in range(len(table)):
            at = lens[r] // page
            if rng.random() < 0.3 and at < width and table[r][at] >= 0:
                refs[table[r][at]] -= 1
                table[r][at] = rng.choice([-1, -1, -(1 << 31)])
        got, want = ops.fork_pages(*on(dev, table, lens, parents, refs), page), plain(table, lens, parents, refs, page)
        for key in KEYS:
            assert getattr(got, key).tolist() == want[key], key


@pytest.mark.parametrize("R,G,pages,width,steps", [(1, 4, 9, 12, 40), (2, 3, 14, 12, 40), (3, 4, 2060, 12, 25)])
def test_tokens_of_a_pool_that_runs_out(dev, R, G, pages, width, steps):
    """Every row's cache holds its own tokens, step after step, while pages run out and become free again."""
    import torch
    from forge_amd import ops
    P = 4
    for seed in range(3):
        say(f"fork_pages, full pools, {R} x {G} of {pages} pages, seed={seed}")
        rng = random.Random(seed)
        taken = max(0, pages - 25)                                   # (held by somebody else)
        refs = [0] * (pages - taken) + [1] * taken
        free = list(range(pages - taken))
        table, rows, lens = [], [], []
        cache = torch.zeros((pages, P), dtype=torch.int32, device=dev)
        for r in range(R * G):
            n = rng.randint(1, 2 * P) if r % G == 0 else 0
            own = [free.pop(0) for _ in range((n + P - 1) // P)]
            for p in own:
                refs[p] = 1
            rows.append([1000 * r + i + 1 for i in range(n)])
            for i, x in enumerate(rows[-1]):
                cache[own[i // P], i % P] = x
            table.append(own + [-1] * (width - len(own)))
            lens.append(n)
        t = on(dev, table, lens, [[0] * G] * R, refs)
        missed = ended = 0
        for step in range(steps):
            was, n0 = t[0].tolist(), t[1].tolist()
            want = plain(was, n0, t[2].tolist(), t[3].tolist(), P)
            got = ops.fork_pages(*t, P)
            for key in KEYS:
                assert getattr(got, key).tolist() == want[key], (step, key)
            ops.copy_pages([cache], got.src, got.dst)
            parents = t[2].flatten().tolist()
            rows = [rows[r // G * G + p][:want["lens"][r]] if 0 <= p < G else [] for r, p in enumerate(parents)]
            ended += sum(lost(was[r // G * G + p], n0[r // G * G + p], P) for r, p in enumerate(parents) if 0 <= p < G)
            for r, s in enumerate(want["slots"]):
                if s >= 0:
                    rows[r].append(100000 * (step + 1) + r)
                    cache[s // P, s % P] = rows[r][-1]
                elif len(rows[r]) % P:
                    missed += 1
            now = cache.tolist()
            lens = [n + (s >= 0) for n, s in zip(want["lens"], want["slots"])]
            for r, n in enumerate(lens):
                if not lost(want["table"][r], n, P):
                    held = [now[want["table"][r][i // P]][i % P] for i in range(n)]
                    assert held == rows[r], (step, r)
            live = [[g for g in range(G) if lens[b * G + g] > 0] or [-1] for b in range(R)]
            parents = [[rng.choice(live[b] + live[b][:1]) for _ in range(G)] for b in range(R)]
            t = [got.table, *on(dev, lens, parents), got.refs]
        assert missed and ended                                      # (the pool did run out)


@pytest.mark.parametrize("end", [None, 3])
@pytest.mark.parametrize("pages,max_len,steps", [(9, 300, 60), (12, 300, 60), (60, 50, 50)])
def test_search_without_room(dev, end, pages, max_len, steps):
    """Searches whose pool or whose table runs out: rows go on from rows all of whose tokens are in the cache, and from ended ones."""
    import torch
    from forge_amd import ops
    from forge_amd.nn import PagedBeams
    B, W, D, page, V = 2, 4, 64, 16, 12
    dropped = after = 0
    for seed in range(3):
        say(f"search without room, {pages} pages, up to {max_len}, end={end} seed={seed}")
        g = torch.Generator().manual_seed(seed)
        kinds = torch.randn((2, V, 1, D), generator=g).to(dev)
        places = torch.randn((2, 300, 1, D), generator=g).to(dev)

        def kv(tokens, at):
            t, p = tokens.long().clamp_min(0), at.long()
            return tuple((kinds[i, t] + places[i, p]).half() for i in range(2))
        prompts = [torch.randint(V, (n,), generator=g).to(dev) for n in (9, 20)]
        lens = [len(p) for p in prompts]
        beams = PagedBeams(B, W, pages, page, max_len, dev)
        cache = torch.zeros(ops.cache4_shape(pages, page, 1, D), dtype=torch.uint8, device=dev)
        slots = beams.start(lens)
        ops.cache4_write(*kv(torch.cat(prompts), torch.cat([torch.arange(n, device=dev) for n in lens])), cache, slots)
        rows = [p.tolist() if w == 0 else None for p in prompts for w in range(W)]
        for step in range(steps):
            logits = (torch.randn((B, W, V), generator=g) * 2).half().to(dev)
            gone = (beams.slots < 0).view(B, W) & ~(beams.ended if end is not None else torch.zeros_like(beams.ended))
            before, ended = beams.scores.clone(), beams.ended.clone()
            if step:
                dropped += int((gone & (before > float("-inf"))).sum())
                before[gone] = float("-inf")
            tokens, parents = beams.step(logits, [cache], end)
            check_selection(logits, before, W, (beams.scores, parents, tokens), None if end is None else ended, end or 0)
            par, tok = parents.tolist(), tokens.tolist()
            rows = [rows[b * W + par[b][w]] + [tok[b][w]] if par[b][w] >= 0 else None for b in range(B) for w in range(W)]
            ops.cache4_write(*kv(tokens.flatten(), beams.lens), cache, beams.slots)
            done = beams.ended.flatten().tolist()
            for r, s in enumerate(beams.slots.tolist()):
                if rows[r] is None or s < 0 or (end is not None and done[r]):
                    continue
                after += dropped > 0
                n = len(rows[r])
                assert beams.lens[r] == n - 1, (step, r)
                at = torch.arange(n, device=dev)
                mine = (beams.table[r, at // page].long() * page + at % page).to(torch.int32)
                for got, want in zip(ops.cache4_read(cache, mine, D), kv(torch.tensor(rows[r], device=dev), at)):
                    assert torch.equal(got, stored(want, D, "float16")), (step, r)
    assert (dropped or end is not None) and (after or max_len < 100)


def test_a_table_that_is_full(dev):
    """The last token needs no slot: its row keeps its score, and is gone with the step after it."""
    import torch
    from forge_amd.nn import PagedBeams
    beams = PagedBeams(1, 2, 20, 16, 20, dev)
    cache = torch.zeros((20, 16), device=dev)
    beams.start([20])
    x = torch.randn((1, 2, 50), generator=torch.Generator().manual_seed(1)).to(dev)
    for step in range(13):
        tokens, parents = beams.step(x, [cache])
        assert (parents >= 0).all() and torch.isfinite(beams.scores).all() and (beams.slots >= 0).all() == (step < 12)
    tokens, parents = beams.step(x, [cache])
    assert (parents == -1).all() and (tokens == -1).all() and (beams.scores == float("-inf")).all() and (beams.lens == 0).all()
