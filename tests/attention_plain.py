"""Attention in 64 bits with its error bound, for the tests of the attention operators."""
import torch

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attention(q, k, v, seen, scale, dtype):
    """(result, bound) of softmax(scale q k^T) v over the seen keys: q (R, D), k and v (n, D), seen (R, n). Only
    seen keys enter, whatever the others hold; a row that sees nothing is zero.

    Bound of a kernel with FP32 scores and sums, weights rounded to `dtype` (relative to the row's largest) and one
    rounding of the result: with u half a unit in the last place and A = sum p |v|,
        u |o| + (u + 2 ds + 2^-20) A + t sum |v| / l,
    ds = (D + 4) 2^-23 max scale sum |q| |k| the largest error of a score, t the smallest step of FP16 weights (0 for BF16)."""
    q, k, v = q.double(), k.double(), v.double()
    R, n = q.shape[0], k.shape[0]
    if n == 0:
        return torch.zeros((R, v.shape[1]), dtype=torch.float64, device=q.device), 0.0
    kz = torch.where(torch.isfinite(k), k, 0.0)
    vz = torch.where(torch.isfinite(v), v, 0.0)
    s = (q @ kz.T) * scale
    mag = ((q.abs() @ kz.abs().T) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(s - top)
    l = p.sum(-1, keepdim=True).clamp_min(1e-300)
    any_seen = seen.any(-1, keepdim=True)
    o = torch.where(any_seen, (p @ vz) / l, 0.0)
    A = (p @ vz.abs()) / l
    u = HALF_ULP[dtype]
    ds = (q.shape[1] + 4) * 2.0 ** -23 * mag
    t = 2.0 ** -24 if dtype == torch.float16 else 0.0
    bound = u * o.abs() + (u + 2 * ds + 2.0 ** -20) * A + t * (seen.double() @ vz.abs()) / l + 2.0 ** -25
    return o, torch.where(any_seen, bound, 0.0)


def check(got, q, k, v, seen, scale):
    o, bound = attention(q, k, v, seen, scale, got.dtype)
    bad = ~((got.double() - o).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound, first at {bad.nonzero()[0].tolist()}"
