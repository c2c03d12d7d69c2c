"""GPU: 4-bit weights (quantize, pack) and int4_linear against plain 64-bit forms.

Bounds: a 16-bit result is off by half a unit in the last place (2^-11 of it for FP16, 2^-8 for BF16); an FP32
sum of n products by at most n 2^-23 of the sum of their magnitudes, where BF16's products are taken with weights
shifted by 136."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu

HALF_ULP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def unpack(w_int4, K):
    """The stored words back to (N, K) integers, from the description of the storage."""
    import torch
    w = w_int4.cpu().to(torch.int64)
    N = w.shape[0]
    words = w.view(N, -1, 4)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    q = torch.empty((N, words.shape[1] * 8), dtype=torch.int64)
    for c in range(words.shape[1]):                      # natural word c of the row
        block, g, j = c // 16, c % 4, c % 16 // 4
        word = words[:, 16 * block + 4 * g + j]
        for e in range(8):
            q[:, 8 * c + e] = (word >> (4 * (e // 2) + 16 * (e % 2)) & 15) - 8
    assert (q[:, K:] == 0).all()
    return q[:, :K]


def check(y, x, q, s, bias, G):
    import torch
    dt = str(x.dtype).split(".")[1]
    xd, qd = x.cpu().double(), q.double()
    sd = s.cpu().double().repeat_interleave(G, 1)
    want = xd @ (qd * sd).T
    mag = xd.abs() @ ((qd.abs() + (272 if dt == "bfloat16" else 0)) * sd).T
    if bias is not None:
        want += bias.cpu().double()
        mag += bias.cpu().double().abs()
    err = (y.cpu().double() - want).abs()
    n = x.shape[1] + 32
    assert y.dtype == x.dtype and torch.isfinite(y).all()
    assert (err <= HALF_ULP[dt] * want.abs() + n * 2.0 ** -23 * mag).all()
    if want.numel() > 1000:
        assert err.norm() <= 1.05 * HALF_ULP[dt] * want.norm()


def make(M, K, N, G, dt, bias, dev, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (N, K), generator=g)
    q[0] = -8
    s = (torch.rand((N, K // G), generator=g) * 1e-2 + 1e-3).half()
    x = torch.randn((M, K), generator=g).to(getattr(torch, dt))
    b = torch.randn((N,), generator=g).to(x.dtype) if bias else None
    return q, s.to(dev), x.to(dev), b.to(dev) if bias else None


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,K,N,G", [
    (1, 32, 1, 32), (1, 128, 17, 128), (3, 64, 16, 64), (1, 4096, 64, 128), (2, 96, 33, 32), (15, 160, 31, 32),
    (16, 2880, 47, 32), (17, 2880, 48, 64), (31, 1152, 130, 128), (33, 416, 15, 32), (64, 640, 257, 64),
    (65, 384, 40, 128), (200, 256, 20, 64), (5, 8192, 40, 128), (48, 6144, 100, 32)])
def test_int4_linear(dev, dt, M, K, N, G):
    linear_case(dev, dt, M, K, N, G)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,K,N,G", [
    (1, 256, 16400, 128), (4, 544, 17001, 32), (7, 288, 8200, 32), (16, 384, 11008, 128), (20, 320, 11001, 64),
    (32, 256, 8193, 32), (40, 416, 12289, 32), (64, 512, 11008, 128), (130, 256, 9000, 64)])
def test_wide_layers(dev, dt, M, K, N, G):
    """Row counts that take the other tiles."""
    linear_case(dev, dt, M, K, N, G)


def linear_case(dev, dt, M, K, N, G):
    from forge_amd import ops
    q, s, x, b = make(M, K, N, G, dt, (M + N) % 2 == 0, dev, M + K + N)
    say(f"int4_linear {dt} M={M} K={K} N={N} G={G}")
    import torch
    w = ops.pack_weight_int4(q.to(torch.int8).to(dev))
    assert (unpack(w, K) == q).all()
    check(ops.int4_linear(x, w, s, b), x, q, s, b, G)


@pytest.mark.parametrize("wdt", ["float16", "float32"])
@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (5, 96, 32), (16, 128, 128), (33, 192, 64), (64, 1024, 128)])
def test_quantize_weight_int4(dev, wdt, N, K, G):
    import torch
    from forge_amd import ops
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn((N, K), generator=g) * 0.05).to(getattr(torch, wdt))
    w[0, :G] = 0.0                                       # an empty group, and one whose scale is below FP16
    if N > 2:
        w[1, :G] = 0.0
        w[1, 0] = 3e-8
    say(f"quantize_weight_int4 {wdt} {N}x{K} G={G}")
    packed, scale = ops.quantize_weight_int4(w.to(dev), G)
    groups = w.float().view(N, K // G, G)
    want_s = (groups.abs().amax(-1) / 7.0).half()
    want_s = torch.where(want_s == 0, torch.tensor(2.0 ** -24, dtype=torch.float16), want_s)
    assert torch.equal(scale.cpu(), want_s)
    want_q = (groups / want_s.float()[..., None]).round().clamp(-8, 7).view(N, K)
    assert (unpack(packed, K) == want_q.long()).all()


def test_special_weights(dev):
    """NaN weights count as zero, an infinite one makes its group's scale infinite, as in quantize_weight_rows."""
    import torch
    from forge_amd import ops
    w = torch.randn((4, 64))
    w[1, 3] = float("nan")
    w[2, 40] = float("inf")
    packed, scale = ops.quantize_weight_int4(w.to(dev), 32)
    q = unpack(packed, 64)
    assert q[1, 3] == 0 and torch.isfinite(scale[1]).all()
    assert torch.isinf(scale[2, 1]) and (q[2, 32:] == 0).all() and torch.isfinite(scale[2, 0])


def test_rows_do_not_mix(dev):
    """A token of NaN and a weight row with an infinite scale leave the others' results as they are; a token's result
    does not depend on how many others there are."""
    import torch
    from forge_amd import ops
    q, s, x, _ = make(16, 512, 48, 128, "float16", False, dev, 1)
    w = ops.pack_weight_int4(q.to(torch.int8).to(dev))
    clean = ops.int4_linear(x, w, s)
    x2, s2 = x.clone(), s.clone()
    x2[5] = float("nan")
    s2[7, 1] = float("inf")
    y = ops.int4_linear(x2, w, s2)
    rows = [m for m in range(16) if m != 5]
    cols = [n for n in range(48) if n != 7]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    assert torch.isnan(y[5]).all() and not torch.isfinite(y[:, 7]).any()
    assert torch.equal(ops.int4_linear(x[:1].contiguous(), w, s), clean[:1])


def test_buffers_and_streams(dev):
    import torch
    from forge_amd import ops
    q, s, x, b = make(4, 1024, 96, 64, "bfloat16", True, dev, 2)
    w = ops.pack_weight_int4(q.to(torch.int8).to(dev))
    want = ops.int4_linear(x, w, s, b)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ops.int4_linear(x, w, s, b, out=out) is out
    side.synchronize()
    assert torch.equal(out, want)
    assert ops.int4_linear(x[:0], w, s, b).shape == (0, 96)


def test_refusals(dev):
    import torch
    from forge_amd import ops
    q, s, x, b = make(4, 256, 32, 64, "float16", True, dev, 3)
    w = ops.pack_weight_int4(q.to(torch.int8).to(dev))
    with pytest.raises(TypeError):
        ops.int4_linear(x.float(), w, s)
    with pytest.raises(TypeError):
        ops.int4_linear(x, w, s, b.to(torch.bfloat16))
    with pytest.raises(TypeError):
        ops.int4_linear(x, w.view(torch.int8), s)
    with pytest.raises(TypeError):
        ops.int4_linear(x, w, s.float())
    with pytest.raises(ValueError):
        ops.int4_linear(x.cpu(), w, s)
    with pytest.raises(ValueError):
        ops.int4_linear(x[:, :192], w, s)               # not contiguous
    with pytest.raises(ValueError):
        ops.int4_linear(x[:, :192].contiguous(), w, s)  # no whole number of groups
    with pytest.raises(ValueError):
        ops.int4_linear(x, w[:, :64].contiguous(), s)
    with pytest.raises(ValueError):
        ops.int4_linear(x, w, s[:, :2].contiguous()[:31])
    with pytest.raises(ValueError):
        ops.int4_linear(x.view(-1)[4:4 + 512].view(2, 256), w, s)   # 8-byte aligned
    with pytest.raises(ValueError):
        ops.int4_linear(x, w, s, out=torch.empty((4, 31), dtype=torch.float16, device=dev))
    with pytest.raises(ValueError):
        ops.quantize_weight_int4(torch.zeros((4, 96), device=dev), 64)
    with pytest.raises(ValueError):
        ops.quantize_weight_int4(torch.zeros((4, 96), device=dev), 96)
    with pytest.raises(TypeError):
        ops.quantize_weight_int4(torch.zeros((4, 64), dtype=torch.int8, device=dev), 32)
    with pytest.raises(ValueError):
        ops.pack_weight_int4(torch.zeros((4, 40), dtype=torch.int8, device=dev))
