"""GPU: qk_norm_rope and its cache form against a plain 64-bit form.

Bound: half a unit in the last place of the 16-bit result, and 2^-20 of the pair's magnitudes for the FP32 steps (some
twenty roundings of 2^-24 and the reciprocal root)."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu

HALF_ULP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def plain(x, w, cos, sin, pos, eps, interleaved):
    """(result, magnitude of the pair) in 64 bits."""
    import torch
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    y, mag = x.clone(), x.abs()
    h = cos.shape[1]
    for i in range(h):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
        c, s = cos[pos, i].double()[:, None], sin[pos, i].double()[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


def close(got, want, dt):
    y, mag = want
    assert ((got.double() - y).abs() <= HALF_ULP[dt] * y.abs() + 2.0 ** -20 * mag + 2.0 ** -25).all()


def make(T, Hq, Hkv, D, R, dt, dev, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    d = getattr(torch, dt)
    qkv = (torch.randn((T, Hq + 2 * Hkv, D), generator=g) * 2).to(d).to(dev)
    w = [(torch.rand((D,), generator=g) + 0.5).to(d).to(dev) for _ in range(2)]
    P = 50
    angle = torch.rand((P, R // 2), generator=g) * 6.0
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32).to(dev)
    return qkv, w, angle.cos().to(dev), angle.sin().to(dev), pos


CASES = [(1, 1, 1, 8, 0), (1, 4, 2, 64, 64), (3, 8, 1, 128, 128), (5, 3, 1, 80, 80), (2, 7, 7, 96, 48), (17, 5, 2, 256, 256),
         (4, 2, 2, 200, 32), (1030, 4, 2, 64, 32), (6, 1, 1, 16, 16), (2, 33, 3, 72, 64)]


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,R", CASES)
def test_qk_norm_rope(dev, T, Hq, Hkv, D, R, interleaved, dt):
    import torch
    from forge_amd import ops
    qkv, (qw, kw), cos, sin, pos = make(T, Hq, Hkv, D, R, dt, dev, T + D + R)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    eps = 1e-5
    say(f"qk_norm_rope {dt} T={T} Hq={Hq} Hkv={Hkv} D={D} R={R} interleaved={interleaved}")
    qo, ko = ops.qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=eps, interleaved=interleaved)
    close(qo, plain(q, qw, cos, sin, pos.long(), eps, interleaved), dt)
    close(ko, plain(k, kw, cos, sin, pos.long(), eps, interleaved), dt)
    # without a norm; only one side normed
    qn, kn = ops.qk_norm_rope(q, k, None, kw, cos, sin, pos, eps=eps, interleaved=interleaved)
    close(qn, plain(q, None, cos, sin, pos.long(), eps, interleaved), dt)
    assert torch.equal(kn, ko)
    # into the cache: rows in any order, one token without a slot, one past the end
    pages, page = (T + 2) // 16 + 2, 16
    slots = torch.randperm(pages * page)[:T].to(torch.int32)
    if T > 2:
        slots[1], slots[2] = -1, pages * page
    kc = torch.full((pages, page, Hkv, D), 7.0, dtype=q.dtype, device=dev)
    vc = torch.full_like(kc, 9.0)
    want_k, want_v = kc.clone().view(-1, Hkv, D), vc.clone().view(-1, Hkv, D)
    ok = (slots >= 0) & (slots < pages * page)
    want_k[slots[ok].long()] = ko[ok.to(dev)]
    want_v[slots[ok].long()] = v[ok.to(dev)]
    qc = ops.qk_norm_rope_cache(q, k, v, qw, kw, cos, sin, pos, kc, vc, slots.to(dev), eps=eps, interleaved=interleaved)
    assert torch.equal(qc, qo)
    assert torch.equal(kc.view(-1, Hkv, D), want_k) and torch.equal(vc.view(-1, Hkv, D), want_v)


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_other_stream(dev, interleaved):
    import torch
    from forge_amd import ops
    qkv, (qw, kw), cos, sin, pos = make(9, 4, 2, 128, 64, "float16", dev, 5)
    q, k = qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous()
    want = ops.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=interleaved)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=interleaved, q_out=q, k_out=k)
    side.synchronize()
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_unknown_positions_and_special_values(dev):
    """Positions outside the table give NaN in the rotated part, an infinite or NaN value spoils its own head only, and
    a head of zeros stays zero."""
    import torch
    from forge_amd import ops
    qkv, (qw, kw), cos, sin, pos = make(6, 3, 1, 64, 32, "bfloat16", dev, 6)
    q, k = qkv[:, :3].contiguous(), qkv[:, 3:4].contiguous()
    clean, _ = ops.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    pos2 = pos.clone()
    pos2[1], pos2[2] = -1, 50
    q2 = q.clone()
    q2[3, 1, 5] = float("nan")
    q2[4, 0, 60] = float("inf")
    q2[5, 2] = 0.0
    got, _ = ops.qk_norm_rope(q2, k, qw, kw, cos, sin, pos2)
    assert torch.isnan(got[1:3, :, :32]).all() and torch.equal(got[1:3, :, 32:], clean[1:3, :, 32:])
    assert torch.isnan(got[3, 1]).all() and torch.equal(got[3, [0, 2]], clean[3, [0, 2]])
    assert torch.equal(got[4, 1:], clean[4, 1:]) and torch.isnan(got[4, 0, 60])
    assert (got[5, 2] == 0).all() and torch.equal(got[0], clean[0])


def test_refusals(dev):
    import torch
    from forge_amd import ops
    qkv, (qw, kw), cos, sin, pos = make(4, 4, 2, 64, 64, "float16", dev, 7)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    f = ops.qk_norm_rope
    with pytest.raises(TypeError):
        f(q.float(), k.float(), qw, kw, cos, sin, pos)
    with pytest.raises(TypeError):
        f(q, k.to(torch.bfloat16), qw, kw, cos, sin, pos)
    with pytest.raises(TypeError):
        f(q, k, qw, kw, cos.half(), sin.half(), pos)
    with pytest.raises(TypeError):
        f(q, k, qw, kw, cos, sin, pos.long())
    for bad in (lambda: f(q.cpu(), k, qw, kw, cos, sin, pos), lambda: f(q, k[:3], qw, kw, cos, sin, pos),
                lambda: f(q[..., :60], k[..., :60], None, None, cos, sin, pos),
                lambda: f(q[..., ::2], k[..., ::2], None, None, cos[:, :16].contiguous(), sin[:, :16].contiguous(), pos),
                lambda: f(q[..., 4:44], k[..., 4:44], None, None, cos[:, :16].contiguous(), sin[:, :16].contiguous(), pos),
                lambda: f(q, k, qw[:32].contiguous(), kw, cos, sin, pos), lambda: f(q, k, qw, kw, cos, sin, pos[:3]),
                lambda: f(q, k, qw, kw, cos[:, :12].contiguous(), sin[:, :12].contiguous(), pos),
                lambda: f(q, k, qw, kw, cos, sin[:10], pos),
                lambda: f(q, k, qw, kw, cos, sin, pos, q_out=torch.empty((4, 3, 64), dtype=q.dtype, device=dev))):
        with pytest.raises(ValueError):
            bad()
    kc = torch.zeros((2, 16, 2, 64), dtype=q.dtype, device=dev)
    slots = torch.zeros((4,), dtype=torch.int32, device=dev)
    g = ops.qk_norm_rope_cache
    for bad in (lambda: g(q, k, v[:, :1], qw, kw, cos, sin, pos, kc, kc.clone(), slots),
                lambda: g(q, k, v, qw, kw, cos, sin, pos, kc[:, :, :1].contiguous(), kc, slots),
                lambda: g(q, k, v, qw, kw, cos, sin, pos, kc, kc[:1], slots),
                lambda: g(q, k, v, qw, kw, cos, sin, pos, kc[:, ::2], kc[:, ::2], slots),
                lambda: g(q, k, v, qw, kw, cos, sin, pos, kc, kc.clone(), slots[:2])):
        with pytest.raises(ValueError):
            bad()
