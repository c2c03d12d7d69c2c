"""GPU: beam_select against a selection in 64 bits. Places are compared exactly; where two scores lie closer than the kernel's own
error (2^-20 of FP32 exponentials and their sums, relative to a sum of about one), either order is right."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu

NEAR = 2.0 ** -20


def plain(logits, scores, count, ended=None, end_token=0):
    """The selection in 64 bits on the host: lists of (score, beam, token), by score and then place; and all scores."""
    import torch
    x = logits.double().cpu()
    B, W, V = x.shape
    prev = scores.double().cpu()
    flat = torch.full((B, W, V), float("-inf"), dtype=torch.float64)
    for b in range(B):
        for w in range(W):
            if ended is not None and ended[b, w]:
                flat[b, w, end_token] = prev[b, w] if torch.isfinite(prev[b, w]) else float("-inf")
                continue
            row = x[b, w]
            ok = torch.isfinite(prev[b, w]) and not row.isnan().any() and not (row == float("inf")).any() and (row > float("-inf")).any()
            if ok:
                row = row - row.max()                 # (first: logits near a type's lowest value are all that 64 bits hold)
                flat[b, w] = row - torch.logsumexp(row, 0) + prev[b, w]
    order = flat.flatten(1).sort(dim=-1, descending=True, stable=True)
    return order.values[:, :count], order.indices[:, :count], flat


def check(logits, scores, count, got, ended=None, end_token=0):
    import torch
    V = logits.shape[2]
    values, at, flat = plain(logits, scores, count, ended, end_token)
    s, w, v = (t.cpu() for t in got)
    assert s.dtype == torch.float32 and w.dtype == v.dtype == torch.int32
    for b in range(logits.shape[0]):
        used = set()
        for i in range(count):
            want = values[b, i].item() if i < values.shape[1] else float("-inf")
            if want == float("-inf"):
                assert (s[b, i].item(), w[b, i].item(), v[b, i].item()) == (float("-inf"), -1, -1), (b, i)
                continue
            place = w[b, i].item() * V + v[b, i].item()
            mine = flat[b].flatten()[place].item()
            room = NEAR + 2.0 ** -50 * abs(want)
            assert place not in used and abs(mine - want) <= room, (b, i, place, at[b, i].item(), mine, want)
            assert abs(s[b, i].item() - mine) <= room + 2.0 ** -24 * abs(mine)
            if place != at[b, i].item():      # another one only where the scores are nearly, and not exactly, equal
                assert mine != want, (b, i, place, at[b, i].item())
            used.add(place)


def logits_of(B, W, V, dt, dev, seed, spread=2.5):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, W, V), generator=g) * spread).to(getattr(torch, dt)).to(dev)


def scores_of(B, W, dev, seed):
    import torch
    return -(torch.rand((B, W), generator=torch.Generator().manual_seed(seed)) * 3).cumsum(-1).to(dev)


def run(dev, dt, B, W, V, count, seed=0, ended=None, end_token=0, logits=None, scores=None):
    import torch
    from forge_amd import ops
    say(f"beam_select {dt} B={B} W={W} V={V} count={count}")
    x = logits_of(B, W, V, dt, dev, seed + V) if logits is None else logits
    s = scores_of(B, W, dev, seed) if scores is None else scores
    got = ops.beam_select(x, s, count, ended=ended, end_token=end_token)
    check(x, s, count, got, ended, end_token)
    return x, s, got


@pytest.mark.parametrize("dt", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("B,W,V,count", [(1, 1, 1, 1), (1, 1, 1, 3), (2, 3, 7, 21), (2, 3, 7, 64), (1, 4, 1000, 8), (3, 5, 2047, 5), (2, 2, 2049, 64),
                                         (1, 16, 8193, 32), (4, 1, 50257, 2), (1, 64, 300, 64), (2, 7, 33001, 14)])
def test_sizes(dev, dt, B, W, V, count):
    run(dev, dt, B, W, V, count)


@pytest.mark.parametrize("dt", ["float16", "float32"])
def test_many_rows(dev, dt):
    """Enough rows for pieces of four vectors a thread."""
    run(dev, dt, 40, 8, 16500, 16)


def test_widest(dev):
    run(dev, "float16", 1, 1024, 50, 64)


@pytest.mark.parametrize("dt", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("V", [100, 2500, 9001])
def test_equal_logits(dev, dt, V):
    """All logits equal, -0 among 0, equal beams: ties go to the lowest (beam, token)."""
    import torch
    x = torch.zeros((2, 3, V), dtype=getattr(torch, dt), device=dev)
    x[:, :, ::3] = -0.0
    s = torch.tensor([[-1.0, -1.0, -2.0], [-3.0, -2.0, -2.0]], device=dev)
    _, _, got = run(dev, dt, 2, 3, V, 40, logits=x, scores=s)
    assert got[1][0].tolist() == [0] * 40 and got[2][0].tolist() == list(range(40))
    assert got[1][1].tolist() == [1] * 40


@pytest.mark.parametrize("dt,B,W,V", [("float16", 2, 64, 300), ("float32", 40, 8, 16500), ("bfloat16", 40, 8, 16500)])
def test_more_equal_than_there_is_room_for(dev, dt, B, W, V):
    """Thousands of candidates with the very same score, in one piece or in one request; with ended beams among them."""
    import torch
    x = torch.full((B, W, V), 1.25, dtype=getattr(torch, dt), device=dev)
    s = torch.full((B, W), -4.0, device=dev)
    _, _, got = run(dev, dt, B, W, V, 64, logits=x, scores=s)
    assert (got[1] == 0).all() and torch.equal(got[2], torch.arange(64, device=dev, dtype=torch.int32).expand(B, 64))
    ended = torch.zeros((B, W), dtype=torch.bool, device=dev)
    ended[:, 1], ended[::2, 3] = True, True
    s[:, 3] = -4.5
    run(dev, dt, B, W, V, 64, logits=x, scores=s, ended=ended, end_token=2)


@pytest.mark.parametrize("V", [501, 4099])
def test_equal_beams(dev, V):
    """Two beams with the same logits, at addresses of different alignment, tie exactly."""
    x = logits_of(1, 1, V, "float16", dev, 5).expand(1, 4, V).contiguous()
    s = scores_of(1, 1, dev, 6).expand(1, 4).contiguous()
    _, _, got = run(dev, "float16", 1, 4, V, 12, logits=x, scores=s)
    assert got[1][0].tolist() == [0, 1, 2, 3] * 3


def test_runs_of_large_neighbours(dev):
    """Orders that put far more above the bound than there is room for: rising logits, a block of large ones, and a whole row
    that is banned but for its end."""
    import torch
    V = 30000
    x = torch.arange(V, device=dev).float()[None, None].repeat(1, 2, 1) * 1e-3
    run(dev, "float32", 1, 2, V, 64, logits=x, scores=torch.zeros((1, 2), device=dev))
    run(dev, "float32", 1, 2, V, 64, logits=-x, scores=torch.zeros((1, 2), device=dev))
    y = logits_of(40, 8, V, "float16", dev, 8)
    y[:, :, 8192:8192 + 2048] += 30.0
    y[:, ::2, : V - 9] = float("-inf")
    run(dev, "float16", 40, 8, V, 64, logits=y)


def test_banned_and_odd_rows(dev):
    import torch
    x = logits_of(4, 4, 3000, "float16", dev, 9)
    x[:, :, 10:2990] = float("-inf")                                 # 20 tokens are left
    x[0, 0] = float("-inf")                                          # none
    x[1, 1, 5] = float("nan")
    x[1, 2, 2995] = float("inf")
    s = scores_of(4, 4, dev, 10)
    s[2, 0], s[2, 1], s[2, 2], s[2, 3] = float("-inf"), float("nan"), float("inf"), -1e30
    s[3] = float("-inf")
    run(dev, "float16", 4, 4, 3000, 64, logits=x, scores=s)
    x[:] = float("-inf")
    _, _, got = run(dev, "float16", 4, 4, 3000, 3, logits=x, scores=scores_of(4, 4, dev, 10))
    assert (got[1] == -1).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("B,W,V,count", [(1, 4, 9001, 8), (1, 2, 20000, 64), (40, 8, 16500, 30)])
def test_masks_of_the_lowest_value(dev, dt, B, W, V, count):
    """A few tokens are allowed and the others hold the type's lowest value, which is a candidate still: thousands of equal ones in
    each piece, of which the first are taken. Then many allowed, and rows of two values."""
    import torch
    d = getattr(torch, dt)
    g = torch.Generator().manual_seed(V)
    full = logits_of(B, W, V, dt, dev, 21)
    for allowed in (0, 3, 20, 500):
        x = torch.full_like(full, torch.finfo(d).min)
        some = torch.randperm(V, generator=g)[:allowed].to(dev)
        x[:, :, some] = full[:, :, some]
        run(dev, dt, B, W, V, count, logits=x)
    run(dev, dt, B, W, V, count, logits=(full > 2.0).to(d))
    run(dev, dt, B, W, V, count, logits=(full > -2.0).to(d) * 3)


@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
@pytest.mark.parametrize("W,V", [(9, 100000), (3, 70000), (40, 9000)])
def test_many_places_of_few_live_beams(dev, dt, W, V):
    """Most lists are empty, so that far more candidates than there is room for reach the first bound."""
    import torch
    ended = torch.ones((2, W), dtype=torch.bool, device=dev)
    ended[:, W // 2] = False
    ended[1, -1] = False
    run(dev, dt, 2, W, V, 60, ended=ended, end_token=11)
    run(dev, dt, 2, W, V, 60)


def test_ended(dev):
    """An ended beam has one candidate, and what its logits hold is not read."""
    import torch
    x = logits_of(3, 4, 900, "bfloat16", dev, 11)
    ended = torch.tensor([[True, False, False, True], [True] * 4, [False] * 4], device=dev)
    s = scores_of(3, 4, dev, 12)
    s[1, 2] = float("-inf")
    x[0, 3], x[1] = float("nan"), float("nan")
    _, _, got = run(dev, "bfloat16", 3, 4, 900, 8, logits=x, scores=s, ended=ended, end_token=899)
    assert got[2][1].tolist() == [899, 899, 899] + [-1] * 5
    run(dev, "bfloat16", 3, 4, 900, 8, logits=x, scores=s, ended=ended, end_token=0)


def test_strides(dev):
    """Rows of any stride and alignment, and a batch that is a transposed view."""
    import torch
    from forge_amd import ops
    for dt in ("float16", "float32"):
        big = logits_of(5, 7, 3001, dt, dev, 13)
        for x in (big[1:4, 2:5, 1:2500], big.transpose(0, 1)[:, :3, 3:], big[:, :1].expand(5, 3, 3001), big[::2, ::3, 7:1000]):
            s = scores_of(x.shape[0], x.shape[1], dev, 14)
            check(x, s, 6, ops.beam_select(x, s, 6))


def test_large_scores(dev):
    """Scores of thousands: the order is taken in 64 bits, where FP32 could not tell neighbours apart."""
    import torch
    x = logits_of(2, 6, 5000, "float16", dev, 15, spread=0.01)
    s = -torch.tensor([[5000.0, 5000.0005, 5000.001, 5000.0015, 5000.002, 5000.0025]] * 2, device=dev)
    run(dev, "float16", 2, 6, 5000, 20, logits=x, scores=s)


def test_buffers_graph_and_stream(dev):
    """Given buffers, another stream, and two graphs that share a workspace, replayed between eager calls."""
    import torch
    from forge_amd import ops
    B, W, V, n = 3, 4, 20011, 8
    x, s, want = run(dev, "float16", B, W, V, n)
    ws = torch.full((ops.beam_select_workspace_size(B, W, V, n),), 0xFF, dtype=torch.uint8, device=dev)
    outs = [(torch.empty((B, n), device=dev), torch.empty((B, n), dtype=torch.int32, device=dev),
             torch.empty((B, n), dtype=torch.int32, device=dev)) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ops.beam_select(x, s, n, workspace=ws, out=outs[0]) is outs[0]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want))
    graphs = []
    for o in outs[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.beam_select(x, s, n, workspace=ws, out=o)
        graphs.append(g)
    for i in range(4):
        x.copy_(logits_of(B, W, V, "float16", dev, 100 + i))
        for g, o in zip(graphs, outs[1:]):
            g.replay()
            torch.cuda.synchronize()
            eager = ops.beam_select(x, s, n)
            assert all(torch.equal(a, b) for a, b in zip(o, eager))
    check(x, s, n, outs[1])


def test_refusals(dev):
    import torch
    from forge_amd import ops
    x, s = logits_of(2, 3, 100, "float16", dev, 1), scores_of(2, 3, dev, 1)
    ended = torch.zeros((2, 3), dtype=torch.bool, device=dev)
    for bad in (dict(count=0), dict(count=65), dict(count=2.0), dict(count=True), dict(scores=s[:1]), dict(logits=x[0]), dict(logits=x.transpose(1, 2)),
                dict(ended=ended[:, :2].contiguous()), dict(ended=ended, end_token=100), dict(ended=ended, end_token=-1), dict(scores=s.cpu()),
                dict(workspace=torch.empty(8, dtype=torch.uint8, device=dev)), dict(out=(s, s.int(), s.int())), dict(logits=x[:, :, :0]),
                dict(logits=x[:1].expand(1, 3, 100).repeat(1, 400, 1), scores=scores_of(1, 1200, dev, 1))):
        with pytest.raises(ValueError):
            ops.beam_select(**dict(dict(logits=x, scores=s, count=4), **bad))
    for bad in (dict(logits=x.double()), dict(scores=s.half()), dict(ended=ended.int())):
        with pytest.raises(TypeError):
            ops.beam_select(**dict(dict(logits=x, scores=s, count=4), **bad))
    assert ops.beam_select(x[:0], s[:0], 4)[1].shape == (0, 4)
