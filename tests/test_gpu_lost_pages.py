"""GPU: pools of pages that run out. A row that found no page to copy its last tokens into ends with the next call, however many
pages are free then; every other row's pages hold its own tokens."""
import random

import pytest

from helpers import say
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
