"""GPU: calls at the edges of a beam search: no rows at all, selections by every path, steps with and without an end, and the
example's scores against each sequence alone."""
import types

import pytest

from helpers import say
from test_gpu_beam_select import NEAR, run
from test_gpu_beams import example  # noqa: F401

pytestmark = pytest.mark.gpu


def test_no_rows(dev):
    """Forking nothing keeps the pages' counts, and a step of no requests is none."""
    import torch
    from forge_amd import ops
    from forge_amd.nn import PagedBeams
    refs = torch.arange(50, dtype=torch.int32, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    for _ in range(3):
        torch.full((50,), 77, dtype=torch.int32, device=dev)         # (what an output would hold that nobody writes)
        got = ops.fork_pages(none.view(0, 4), none, none.view(0, 3), refs, 16)
        assert torch.equal(got.refs, refs) and got.table.shape == (0, 4) and got.slots.shape == (0,)
    out = ops.Forked(got.table, none, torch.full_like(refs, -3), none, none, none)
    assert ops.fork_pages(none.view(0, 4), none, none.view(0, 3), refs, 16, workspace=torch.empty(0, dtype=torch.uint8, device=dev), out=out) is out
    assert torch.equal(out.refs, refs)
    beams = PagedBeams(0, 3, 50, 16, 40, dev)
    assert beams.start([]).shape == (0,)
    tokens, parents = beams.step(torch.zeros((0, 3, 9), device=dev), {0: torch.zeros((50, 4), device=dev)}.values(), 2)
    assert tokens.shape == parents.shape == (0, 3) and (beams.refs == 0).all()


@pytest.mark.parametrize("dt,B,W,V,per,piece", [("float16", 40, 8, 16500, 8, 8192), ("bfloat16", 40, 8, 16384, 8, 8192), ("float32", 40, 8, 20000, 4, 8192),
                                                ("float16", 1, 4, 9001, 8, 2048), ("bfloat16", 2, 1, 2048, 8, 2048)])
@pytest.mark.parametrize("count", [64, 63])
def test_a_low_group(dev, dt, B, W, V, per, piece, count):
    """64 places, and of each 64 vectors of a piece one that holds low logits only: its largest is the first bound, and thousands lie above it."""
    import torch
    g = torch.Generator().manual_seed(V + count)
    x = (torch.randn((B, W, V), generator=g) * 2.5).to(getattr(torch, dt))
    low = (torch.arange(V) % piece) // per % 64
    few = low == 17 if count == 64 else (low == 17) | (low == 40)
    x[:, :, few] = (-25.0 - 5.0 * torch.rand((B, W, int(few.sum())), generator=g)).to(x.dtype)
    x[:, :, 5::97] = float("-inf")
    x[0, :, 1000:1040] = 12.0                                        # equal ones at the top
    x[-1, 0] = x[-1, 0].sort(descending=True).values.float().view(-1).to(x.dtype)
    x[-1, 0, few] = -28.0
    run(dev, dt, B, W, V, count, logits=x.to(dev))


@pytest.mark.parametrize("B,W,V,low", [(1, 1024, 64, 64), (2, 1024, 100, 128), (1, 1000, 300, 64), (3, 16, 4000, 8), (1, 512, 200, 64)])
def test_many_rounds(dev, B, W, V, low):
    """Far more candidates above the first bounds than there is room for, as beams in a fixed stride have low scores; near scores and equal
    ones among them."""
    import torch
    g = torch.Generator().manual_seed(W + V)
    for kind in range(4):
        x = torch.randn((B, W, V), generator=g) * (0.01 if kind == 1 else 1.0)
        if kind == 2:
            x = x.round()
        s = torch.rand((B, W), generator=g) * (0.0 if kind == 3 else 1e-2)
        s[:, 3::low] -= 30.0
        run(dev, "float32" if kind < 2 else "float16", B, W, V, 64, logits=x.to(torch.float32 if kind < 2 else torch.float16).to(dev), scores=s.to(dev))


def test_steps_with_and_without_an_end(dev):
    """A step without an end_token lets every row go on; what it leaves at a row's place is not the one that had ended there."""
    import torch
    from forge_amd.nn import PagedBeams
    beams = PagedBeams(2, 3, 60, 16, 40, dev)
    cache = torch.zeros((60, 4), device=dev)
    beams.start([3, 20])
    x = torch.full((2, 3, 9), -20.0, device=dev)
    x[:, :, 2], x[:, :, 4], x[:, :, 5] = 1.0, 0.5, 0.0              # each row: 2 before 4 before 5
    tokens, _ = beams.step(x, [cache], 2)
    assert tokens.tolist() == [[2, 4, 5]] * 2 and beams.ended.tolist() == [[True, False, False]] * 2
    beams.step(x, [cache])
    assert not beams.ended.any()
    before = beams.lens.tolist()
    x[:, :, 2] = -20.0
    tokens, parents = beams.step(x, [cache], 2)                      # (as live rows all of them get 4 or 5)
    assert (tokens != 2).all() and not beams.ended.any()
    assert beams.lens.tolist() == [before[b * 3 + p] + 1 for b in range(2) for p in parents[b].tolist()]
    beams.start([3, 20])
    tokens, _ = beams.step(x, [cache], 4)
    assert beams.ended.any()
    beams.start([3, 20])
    assert not beams.ended.any()


@pytest.mark.parametrize("lens,width,steps,end", [((37, 5, 130), 4, 12, 7), ((16, 1, 31), 5, 40, None), ((64,), 7, 30, 3)])
def test_example_scores(dev, example, lens, width, steps, end):  # noqa: F811
    """Every sequence that the example's search returns, run again in a row of its own: pages in order that no other row names, a copy of the
    prompt's, no selection and no fork. The calls have the same sizes, and a row's result is not its neighbours' matter (fewer keys than
    are split), so the logits are the same, and the scores but for a selection's error and FP32's rounding in each step."""
    import torch
    from forge_amd import ops
    say(f"the example's search of {lens}, {width} beams, {steps} steps, end={end}")
    page = 16
    model = example.Decoder()
    torch.manual_seed(len(lens))
    prompts = [torch.randint(1000, (n,)).tolist() for n in lens]
    found, scores = example.search(model, prompts, width, steps, end, page)
    B, R = len(lens), len(lens) * width
    each = (max(lens) + steps) // page + 1                           # pages of a row, and of a prompt
    of = torch.arange(B).repeat_interleave(width)                    # a row's prompt
    table = torch.arange(R * each, dtype=torch.int32, device=dev).view(R, each)
    whole, caches = model.caches(B * each, page), model.caches(R * each, page)
    at = [torch.arange(n, dtype=torch.int32) for n in lens]
    cu = torch.tensor([0, *lens], device=dev).cumsum(0).to(torch.int32)
    logits = model.prompt(torch.tensor(sum(prompts, []), device=dev), cu, torch.cat(at).to(dev), whole,
                          torch.cat([b * each * page + p for b, p in enumerate(at)]).to(dev))
    logits = logits[(cu[1:] - 1).long()][of.to(dev)]
    for a, b in zip(caches, whole):
        a.view(R, each, -1).copy_(b.view(B, each, -1)[of.to(dev)])
    n = torch.tensor(lens, dtype=torch.int32)[of].to(dev)
    total = torch.zeros(R, dtype=torch.float64, device=dev)
    ended = torch.zeros(R, dtype=torch.bool, device=dev)
    tokens = found.view(R, steps)
    assert (tokens >= 0).all() and torch.isfinite(scores).all()
    for i in range(steps):
        t = tokens[:, i].contiguous()
        gain = torch.log_softmax(logits.double(), -1).gather(1, t.long()[:, None])[:, 0]
        total += torch.where(ended, 0.0, gain)
        if end is not None:
            assert (t[ended] == end).all()
            ended |= t == end
        slots = table.gather(1, (n // page).long()[:, None])[:, 0] * page + n % page
        logits = model.next(t, caches, types.SimpleNamespace(lens=n, slots=slots.to(torch.int32), table=table))
        n = n + 1
    room = steps * (NEAR + 2.0 ** -24 * scores.abs().max().item())
    worst = (total.view(B, width) - scores.double()).abs().max().item()
    assert worst <= room, (worst, room)
    assert len({tuple(x) for x in tokens.tolist()}) == R             # no sequence twice
