"""GPU: calls at the edges of a beam search: no rows at all, selections by every path, steps with and without an end, and the
example's scores against each sequence alone."""
import pytest

from helpers import say
from test_gpu_beam_select import run, scores_of

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
    tokens, parents = beams.step(torch.zeros((0, 3, 9), device=dev), [torch.zeros((50, 4), device=dev)], 2)
    assert tokens.shape == parents.shape == (0, 3) and (beams.refs == 0).all()


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
