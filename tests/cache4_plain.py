"""The 4-bit cache in plain torch, from its definition: quantization, layout, and attention in 64 bits with its error bound."""
import torch

from attention_plain import HALF_ULP

SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]


def units(D):
    return next(u for u in (2, 3, 4, 6, 8) if D <= 32 * u)


def quantize(x):
    """(.., D) of 16 bits -> integers, step and lowest value, in 64 bits (NaN for heads that are not finite)."""
    dt = x.dtype
    x = x.double().cpu()
    low, top = x.amin(-1), x.amax(-1)
    # FP32 quotients, correctly rounded, and their FP32 difference
    want = (top / 15.0).float() - (low / 15.0).float()
    step = want.to(dt)
    step = torch.where(step.float() > want, (step.view(torch.int16) - 1).view(dt), step).double()
    safe = torch.where(step > 0, step, 1.0)[..., None]
    n = torch.where(step[..., None] > 0, ((x - low[..., None]) / safe).float().round().double(), 0.0).clamp(0.0, 15.0)
    odd = ~torch.isfinite(x).all(-1)
    return torch.where(odd[..., None], 0.0, n), step.masked_fill(odd, float("nan")), low.masked_fill(odd, float("nan"))


def held(x):
    """What a cache holds of x (.., D): (values in 64 bits, m + 8 s, s |n - 8| and the steps), on x's device."""
    n, step, low = quantize(x)
    to = lambda t: t.to(x.device)                                    # noqa: E731
    return (to(low[..., None] + n * step[..., None]), to((low + 8 * step)[..., None].expand_as(n).clone()),
            to((n - 8).abs() * step[..., None]), to(step), to(n * step[..., None]), to(low))


def words(cache, page, D):
    """Integers and numbers of a cache by its documented layout: keys and values (pages, heads, page, D) and four
    numbers (pages, heads, page, 4) as int16 bits."""
    W = 4 * units(D)
    flat = cache.cpu().flatten(2)
    shape = flat.shape[:2]
    word = flat[..., :page * 8 * W].contiguous().view(torch.int32).long() & 0xFFFFFFFF
    k = word[..., :page * W].view(*shape, page, W)
    v = word[..., page * W:].view(*shape, page // 4, W, 4).transpose(3, 4).reshape(*shape, page, W)

    def unpack(w):
        return ((w[..., None] >> torch.tensor(SHIFTS)) & 15).flatten(-2)
    num = flat[..., page * 8 * W:].contiguous().view(torch.int16).view(*shape, page, 4)
    return unpack(k), unpack(v), num


def attention(q, k, v, seen, scale, dtype):
    """(result, bound) of cache4_attention for rows q (R, D) over held k and v (held()'s tuples, (n, D)), seen (R, n).

    With u half a unit in the last place of `dtype` and w = p s':
      the result's rounding u |o|; the weights' 2^-11 w |n' - 8| each, or 2^-29 of the row's largest w (half of FP16's
      smallest step, the largest being at 2^4 or above);
      the matrix unit: of the 8 products of a group 7 may lose 2^-18 of the group's largest factor beside the integers (those
      are FP16 subnormals n 2^-20, whose exponent counts as 2^-14, and 24 bits are kept), and a group's products next to each
      other 2^-21 of themselves. Scores, of D / 8 groups, then miss
      ds = 7 2^-18 scale s sum over groups of max |q| + (D / 8 + 12) 2^-23 scale (s sum |q| n + |m| sum |q|) (2^-23 for each
      group's addition, or half of it for the D / 4 of a lane's sum of q, and the few of steps and lowest values), which moves a weight by 2 ds of itself; the sum of w n'
      misses 7 2^-18 of the sum of w, and (keys / 8 + 16) 2^-23 of itself and of 8 times the sum of w, which is taken off;
      the other FP32 sums: (keys / 4 + 64) 2^-23 of what they sum, 2^-18 for the exponentials and factors."""
    q = q.double()
    val_k, _, _, step_k, up_k, low_k = k
    val_v, mid_v, off_v, step_v, up_v, _ = v
    R, n = q.shape[0], val_k.shape[0]
    if n == 0:
        return torch.zeros((R, val_v.shape[1]), dtype=torch.float64, device=q.device), 0.0
    fix = lambda t: torch.nan_to_num(t, nan=0.0)                     # noqa: E731  (unseen ones; a seen NaN is the caller's)
    val_k, up_k, low_k = fix(val_k), fix(up_k), fix(low_k)
    val_v, mid_v, off_v, step_v, up_v = fix(val_v), fix(mid_v), fix(off_v), fix(step_v), fix(up_v)
    s = ((q @ val_k.T) * scale).masked_fill(~seen, float("-inf"))
    mag = ((q.abs() @ up_k.T + q.abs().sum(-1, keepdim=True) * low_k.abs()) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
    l = p.sum(-1, keepdim=True).clamp_min(1e-300)
    any_seen = seen.any(-1, keepdim=True)
    o = torch.where(any_seen, (p @ val_v) / l, 0.0)
    w = p @ off_v / l
    A = (p @ (mid_v.abs() + off_v)) / l
    most = (p * step_v).amax(-1, keepdim=True) / l
    u = HALF_ULP[dtype]
    D = q.shape[1]
    group = q.abs().view(R, D // 8, 8).amax(-1).sum(-1, keepdim=True)
    ds = 7 * 2.0 ** -18 * scale * group * fix(step_k).max() + (D / 8 + 12) * 2.0 ** -23 * mag
    W, S = (p @ up_v) / l + 8 * (p @ step_v)[:, None] / l, (p @ step_v)[:, None] / l
    bound = u * o.abs() + 2.0 ** -11 * w + 2.0 ** -29 * 8 * n * most + (2 * ds + 2.0 ** -18 + (n / 4 + 64) * 2.0 ** -23) * A
    bound = bound + 7 * 2.0 ** -18 * S + (n / 8 + 16) * 2.0 ** -23 * W
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    return o, torch.where(any_seen, bound * (1 + u), 0.0)


def check(got, q, k, v, seen, scale):
    o, bound = attention(q, k, v, seen, scale, got.dtype)
    bad = ~((got.double() - o).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[tuple(bad.nonzero()[0])].item()} for {o[tuple(bad.nonzero()[0])].item()}"
