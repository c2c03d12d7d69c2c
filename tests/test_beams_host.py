"""CPU: what PagedBeams refuses, and what a refused call leaves."""
import pytest


def beams(**more):
    from forge_amd.nn import PagedBeams
    return PagedBeams(**dict(dict(requests=2, beams=3, pages=10, page_size=4, max_len=20, device="cpu"), **more))


def test_refused_step():
    """A step that raises (here for lack of a device) changes nothing, so that it can be made again with what is right."""
    import torch
    b = beams()
    b.start([5, 8])
    b.slots, b._written = torch.tensor([5, -1, -1, 12, -1, -1], dtype=torch.int32), True
    was = {k: v.clone() for k, v in vars(b).items() if isinstance(v, torch.Tensor)}
    for end in (None, 7):
        with pytest.raises(ValueError, match="device"):
            b.step(torch.zeros((2, 3, 9)), [torch.zeros((10, 4))], end)
        assert all(torch.equal(v, getattr(b, k)) for k, v in was.items()) and b._written


def test_other_pages():
    """Caches of another page count than the rows' are refused: with fewer pages, copies would be left out without a word."""
    import torch
    b = beams()
    b.start([5, 8])
    for pages in (9, 11):
        with pytest.raises(ValueError, match="pages"):
            b.step(torch.zeros((2, 3, 9)), [torch.zeros((pages, 4)), torch.zeros((10, 4))])
        with pytest.raises(ValueError, match="pages"):
            b.step(torch.zeros((2, 3, 9)), {0: torch.zeros((pages, 4))}.values())
    with pytest.raises(ValueError, match="device"):                  # (as far as the operators)
        b.step(torch.zeros((2, 3, 9)), (torch.zeros((10, 4)) for _ in range(2)))


def test_limits():
    """What the operators of a step refuse is refused at once."""
    beams(beams=64)
    beams(requests=128, beams=64)
    assert beams(requests=0).start([]).shape == (0,)
    for bad in (dict(beams=65), dict(beams=0), dict(requests=129, beams=64), dict(requests=-1), dict(pages=0)):
        with pytest.raises(ValueError):
            beams(**bad)


def test_start_keeps_results():
    """The scores that a search has left are the caller's: the next start() makes others."""
    import torch
    b = beams()
    b.start([5, 8])
    b.scores, b.ended = torch.full((2, 3), -2.5), torch.ones((2, 3), dtype=torch.bool)
    scores, ended = b.scores, b.ended
    b.start([1, 2])
    assert (scores == -2.5).all() and ended.all()
    assert b.scores.tolist() == [[0.0, float("-inf"), float("-inf")]] * 2 and not b.ended.any()
