"""GPU: the decoder operators at the ends of their ranges: the largest and smallest values, infinities and NaN, empty
and extreme sizes, arguments that are no numbers."""
import pytest

from helpers import say

pytestmark = pytest.mark.gpu


def normals(shape, dt, dev, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(getattr(torch, dt)).to(dev)


# ---- int4_linear ---------------------------------------------------------------------------------

def test_no_values_is_refused(dev):
    """K = 0 has no scale group: an error, not an output that nobody wrote."""
    import torch
    from forge_amd import ops
    x = torch.empty((2, 0), dtype=torch.float16, device=dev)
    w = torch.empty((8, 0), dtype=torch.uint8, device=dev)
    for groups in (0, 1, 3):
        with pytest.raises(ValueError):
            ops.int4_linear(x, w, torch.ones((8, groups), dtype=torch.float16, device=dev))


def int4_case(M, K, N, dt, dev, seed):
    """x, and weights of one scale group whose rows 0 and 1 hold no zero."""
    import torch
    from forge_amd import ops
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (N, K), generator=g)
    q[:2] = torch.where(q[:2] == 0, 3, q[:2])
    s = (torch.rand((N, K // 32), generator=g) * 1e-2 + 1e-3).half().to(dev)
    x = torch.randn((M, K), generator=g).to(getattr(torch, dt)).to(dev)
    return x, q.to(dev), s, ops.pack_weight_int4(q.to(torch.int8).to(dev))


SIZES = [(1, 128, 20), (3, 512, 40), (1, 1024, 16400), (16, 512, 20), (16, 512, 11008), (30, 512, 40), (30, 256, 8200), (64, 512, 50),
         (64, 512, 11008)]


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_int4_infinite_tokens(dev, M, K, N, dt):
    """An infinite activation times a weight of zero is NaN, times any other an infinity, as in the sum of products."""
    import torch
    from forge_amd import ops
    x, q, s, w = int4_case(M, K, N, dt, dev, K + N)
    x[M - 1, 37] = float("inf")
    x[M // 2, K - 2] = float("-inf")
    say(f"int4_linear infinities {dt} M={M} K={K} N={N}")
    y = ops.int4_linear(x, w, s)
    sign = torch.ones((M, N), device=dev)
    hit = torch.zeros((M, N), dtype=torch.bool, device=dev)
    nan = torch.zeros((M, N), dtype=torch.bool, device=dev)
    for m, k, v in ((M - 1, 37, 1.0), (M // 2, K - 2, -1.0)):
        here = v * q[:, k].sign().float()
        nan[m] |= (here == 0) | (hit[m] & (here != sign[m]))
        sign[m] = here
        hit[m] = True
    assert torch.equal(torch.isnan(y), nan)
    assert torch.equal(torch.isinf(y), hit & ~nan)
    assert (y[hit & ~nan].sign() == sign[hit & ~nan]).all()


@pytest.mark.parametrize("M,K,N", SIZES)
def test_int4_large_tokens(dev, M, K, N):
    """BF16 values far above what a shifted weight could take: the sum of products itself stays in range.
    Bound as in test_gpu_int4.py, of products of |q| <= 8: 2^-8 of the result and n 2^-23 of the products' magnitudes."""
    import torch
    from forge_amd import ops
    x, q, s, w = int4_case(M, K, N, "bfloat16", dev, K + N + 1)
    x[:, 5] = 1e37
    x[:, 70] = -1e37
    x[M // 2] = 3e36
    say(f"int4_linear large values M={M} K={K} N={N}")
    y = ops.int4_linear(x, w, s).double()
    ws = q.double() * s.double().repeat_interleave(32, 1)
    want, mag = x.double() @ ws.T.contiguous(), x.double().abs() @ ws.abs().T.contiguous()
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + (K + 32) * 2.0 ** -23 * mag).all()


def int4_bound(x, q, s):
    """The result in 64 bits, and what a kernel with FP32 sums of these products may be off by."""
    ws = q.double() * s.double().repeat_interleave(32, 1)
    want, mag = x.double() @ ws.T.contiguous(), x.double().abs() @ ws.abs().T.contiguous()
    u = 2.0 ** -11 if str(x.dtype) == "torch.float16" else 2.0 ** -8
    return want, u * want.abs() + (x.shape[1] + 32) * 2.0 ** -23 * mag


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,K,N", [(257, 384, 40), (1025, 256, 60), (4099, 128, 17), (300, 512, 8200), (700, 544, 2881)])
def test_int4_prompts(dev, M, K, N, dt):
    """Tokens of whole prompts: many tiles of 64, and rows of fewer values than a unit."""
    from forge_amd import ops
    x, q, s, w = int4_case(M, K, N, dt, dev, M)
    say(f"int4_linear prompt {dt} M={M} K={K} N={N}")
    want, bound = int4_bound(x, q, s)
    assert ((ops.int4_linear(x, w, s).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
def test_int4_one_token_among_others(dev, dt):
    """A token's sums are taken in another order alone than with 15, 31 or 63 others: within the bound, not bit for bit."""
    import torch
    from forge_amd import ops
    x, q, s, w = int4_case(64, 4096, 3000, dt, dev, 5)
    want, bound = int4_bound(x, q, s)
    for M in (1, 4, 5, 16, 17, 32, 33, 64):
        y = ops.int4_linear(x[:M].contiguous(), w, s)
        assert ((y.double() - want[:M]).abs() <= bound[:M]).all()
        assert torch.equal(ops.int4_linear(x[:M].contiguous(), w, s), y)


# ---- qk_norm_rope --------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,e", [(64, 61), (128, 64), (256, 100), (80, 126)])
def test_norm_of_large_heads(dev, D, e, interleaved):
    """Heads of BF16 values whose squares FP32 does not hold are normed as any others; an infinity gives NaN in its own pair
    and zeros elsewhere, as x / inf does. Bound: a head's size and its product with the weight, and the turn, each rounded in
    FP32, then to BF16: 2^-8 of the result and 2^-20 of the pair."""
    import torch
    from forge_amd import ops
    T, Hq, Hkv = 33, 5, 2
    q, k = (normals((T, h, D), "float32", dev, D + h) for h in (Hq, Hkv))
    q[::2] *= 2.0 ** e
    k[1::3] *= 2.0 ** e
    q, k = q.clamp(-3e38, 3e38).to(torch.bfloat16), k.clamp(-3e38, 3e38).to(torch.bfloat16)
    w = (normals((D,), "float32", dev, 1).abs() + 0.5).to(torch.bfloat16)
    R = D // 2 // 16 * 16
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    angle = torch.rand((T, R // 2), device=dev) * 6.0
    cos, sin = angle.cos(), angle.sin()
    qo, ko = ops.qk_norm_rope(q, k, w, w, cos, sin, pos, interleaved=interleaved)
    for x, got in ((q, qo), (k, ko)):
        y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        first = torch.arange(R // 2, device=dev) * (2 if interleaved else 1)
        second = first + (1 if interleaved else R // 2)
        a, b, c, s = y[..., first], y[..., second], cos.double()[:, None], sin.double()[:, None]
        want, size = y.clone(), y.abs()
        want[..., first], want[..., second] = a * c - b * s, b * c + a * s
        size[..., first] = size[..., second] = a.abs() + b.abs()
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 1e-37).all()
    q[3, 1, D - 1] = float("inf")
    qo = ops.qk_norm_rope(q, k, w, w, cos, sin, pos, interleaved=interleaved)[0]
    assert torch.isnan(qo[3, 1, D - 1]) and (qo[3, 1, :D - 2 * (R == D) - 1] == 0).all()
    assert torch.isfinite(qo[3, [0, 2, 3, 4]]).all()


# ---- arguments -----------------------------------------------------------------------------------

class NoBool:
    def __bool__(self):
        raise RuntimeError("no truth value")


@pytest.mark.parametrize("eps,interleaved", [("small", False), (None, False), (1e-6, NoBool())])
def test_bad_numbers_touch_nothing(dev, eps, interleaved):
    """An eps or a flag that is no number is refused before the queries (in place here) or the cache are written."""
    import torch
    from forge_amd import ops
    T, D = 4, 64
    q, k, v = (torch.randn((T, 2, D), device=dev).half() for _ in range(3))
    kc, vc = (torch.randn((2, 16, 2, D), device=dev).half() for _ in range(2))
    cos, sin = torch.rand((8, D // 2), device=dev), torch.rand((8, D // 2), device=dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    w = torch.ones((D,), dtype=torch.float16, device=dev)
    was = [t.clone() for t in (q, kc, vc)]
    with pytest.raises(Exception):
        ops.qk_norm_rope_cache(q, k, v, w, w, cos, sin, pos, kc, vc, pos, eps=eps, interleaved=interleaved, q_out=q)
    torch.cuda.synchronize()
    for t, before in zip((q, kc, vc), was):
        assert torch.equal(t, before)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    out = torch.full_like(q, 5.0)
    with pytest.raises(Exception):
        ops.prompt_attention(q, k, v, cu, causal=NoBool(), out=out)
    torch.cuda.synchronize()
    assert (out == 5.0).all()


def test_heads_of_no_values_are_refused(dev):
    import torch
    from forge_amd import ops
    q = torch.empty((4, 2, 0), dtype=torch.float16, device=dev)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, q, q, cu)
    w = torch.empty((0,), dtype=torch.float16, device=dev)
    table = torch.empty((4, 0), device=dev)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, q, w, w, table, table, cu.new_zeros(4))
    with pytest.raises(ValueError):
        ops.prompt_attention(q.new_zeros(()), q, q, cu)
    cache = torch.empty((1, 16, 2, 0), dtype=torch.float16, device=dev)
    one = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    ws = torch.empty((16,), dtype=torch.uint8, device=dev)
    q4 = q.view(1, 4, 2, 0)
    with pytest.raises(ValueError):
        ops.cache_attention(q4, cache, cache, one, one[0], workspace=ws, out=torch.empty_like(q4))


# ---- attention -----------------------------------------------------------------------------------

def prompt(q, k, v, **kw):
    """prompt_attention of one sequence: q (n, Hq, D), k and v (n, Hkv, D)."""
    import torch
    from forge_amd import ops
    return ops.prompt_attention(q, k, v, torch.tensor([0, q.shape[0]], dtype=torch.int32, device=q.device), **kw)


def cached(q, k, v, T, page=16, tree=None):
    """cache_attention of the last T tokens of one sequence over the others' keys and values: (T, Hq, D)."""
    import torch
    from forge_amd import ops
    n, Hkv, D = k.shape
    pages = (n + page - 1) // page
    kc, vc = (torch.zeros((pages * page, Hkv, D), dtype=k.dtype, device=k.device) for _ in range(2))
    kc[:n], vc[:n] = k, v
    table = torch.arange(pages, dtype=torch.int32, device=k.device)[None]
    lens = torch.tensor([n - T], dtype=torch.int32, device=k.device)
    return ops.cache_attention(q[None, n - T:].contiguous(), kc.view(pages, page, Hkv, D), vc.view(pages, page, Hkv, D), table, lens,
                               tree=tree)[0]


# (tokens, Hq, Hkv, D): every way in which a prompt's rows and keys are split
PROMPTS = [(200, 4, 2, 64), (300, 2, 1, 64), (300, 2, 1, 80), (300, 2, 2, 128), (700, 64, 8, 128), (300, 3, 1, 256)]
# (keys, T, Hq, Hkv, D): one, two and four sets of rows, one chunk of keys and several
CACHES = [(40, 1, 4, 1, 64), (900, 1, 8, 2, 128), (900, 5, 16, 2, 64), (700, 61, 4, 1, 128), (900, 3, 2, 1, 256), (500, 40, 4, 1, 256),
          (2500, 16, 4, 2, 80)]


@pytest.mark.parametrize("dt,top,step", [("bfloat16", -1.0, -1.0), ("bfloat16", -512.0, -512.0), ("bfloat16", 64.0, -1.0),
                                         ("float16", 3.0, -0.25), ("float16", -0.5, -0.25)])
def test_scores_far_from_zero(dev, dt, top, step):
    """Scores of any size that FP32 holds, far apart from key to key: a row's result is the value of its best key. In units of the largest
    scores tried, q k is top + step * (the key's rank)."""
    import torch
    q_one = 1e16 if dt == "bfloat16" else 3e4
    k_one = 1e16 if dt == "bfloat16" else 5e3
    for i, (n, T, Hq, Hkv, D) in enumerate([(n, 0, *rest) for n, *rest in PROMPTS] + CACHES):
        say(f"scores far from zero {dt} top={top} n={n} T={T} Hq={Hq} D={D}")
        v = normals((n, Hkv, D), dt, dev, i)
        q = torch.full((n, Hq, D), q_one, dtype=v.dtype, device=dev)
        rank = torch.randperm(n, generator=torch.Generator().manual_seed(i)) % 8      # 8 different scores, the first keys not the best
        best = torch.tensor([int(rank[:r + 1].min()) for r in range(n)])
        k = ((top + step * rank.float()) * k_one).to(v.dtype).to(dev)[:, None, None].expand(n, Hkv, D).contiguous()
        out = prompt(q, k, v) if T == 0 else cached(q, k, v, T)
        for r in range(n - T if T else 0, n, 1 if T else 7):
            ties = (rank[:r + 1] == best[r]).to(dev)
            mean = v[:r + 1][ties].double().mean(0).repeat_interleave(Hq // Hkv, 0)
            size = v[:r + 1][ties].double().abs().mean(0).repeat_interleave(Hq // Hkv, 0)
            u = 2.0 ** -8 if dt == "bfloat16" else 2.0 ** -11
            got = out[r - (n - T) if T else r].double()
            assert ((got - mean).abs() <= u * mean.abs() + n * 2.0 ** -23 * size + 2.0 ** -25).all(), (r, best[r])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,Hq,Hkv,D", PROMPTS)
def test_largest_values_prompt(dev, n, Hq, Hkv, D, causal):
    """Means of BF16 values whose sum FP32 does not hold."""
    import torch
    from attention_plain import check
    say(f"largest values, prompt n={n} Hq={Hq} D={D} causal={causal}")
    q, k, v = normals((n, Hq, D), "bfloat16", dev, 1), normals((n, Hkv, D), "bfloat16", dev, 2), normals((n, Hkv, D), "bfloat16", dev, 3)
    big = torch.finfo(torch.bfloat16).max
    v = (v.sign().float() * big * (1.0 - 0.6 * torch.rand(v.shape, device=dev))).to(torch.bfloat16)
    v[:, :, 0] = big
    v[:, :, 1] = -big
    out = prompt(q, k, v, causal=causal)
    i = torch.arange(n, device=dev)
    seen = i[None] <= i[:, None] if causal else torch.ones((n, n), dtype=torch.bool, device=dev)
    for h in range(0, Hq, max(1, Hq // 4)):
        g = h // (Hq // Hkv)
        check(out[:, h], q[:, h], k[:, g], v[:, g], seen, D ** -0.5)
    assert (out[:, :, 0] == big).all() and (out[:, :, 1] == -big).all()


@pytest.mark.parametrize("n,T,Hq,Hkv,D", CACHES)
def test_largest_values_cache(dev, n, T, Hq, Hkv, D):
    import torch
    from attention_plain import check
    say(f"largest values, cache n={n} T={T} Hq={Hq} D={D}")
    q, k, v = normals((n, Hq, D), "bfloat16", dev, 4), normals((n, Hkv, D), "bfloat16", dev, 5), normals((n, Hkv, D), "bfloat16", dev, 6)
    big = torch.finfo(torch.bfloat16).max
    v = (v.sign().float() * big * (1.0 - 0.6 * torch.rand(v.shape, device=dev))).to(torch.bfloat16)
    v[:, :, 0] = big
    out = cached(q, k, v, T)
    i = torch.arange(n, device=dev)
    seen = i[None] <= i[n - T:, None]
    for h in range(Hq):
        g = h // (Hq // Hkv)
        check(out[:, h], q[n - T:, h], k[:, g], v[:, g], seen, D ** -0.5)
    assert (out[:, :, 0] == big).all()


@pytest.mark.parametrize("e", [-60, -100, -110])
def test_smallest_values(dev, e):
    """Means of BF16 values near the lower end of its range keep their bits."""
    import torch
    for i, (n, T, Hq, Hkv, D) in enumerate([(n, 0, *rest) for n, *rest in PROMPTS] + CACHES):
        say(f"smallest values 2^{e} n={n} T={T} Hq={Hq} D={D}")
        q, k = normals((n, Hq, D), "bfloat16", dev, i), normals((n, Hkv, D), "bfloat16", dev, i + 1)
        v = torch.full((n, Hkv, D), 2.0 ** e, dtype=torch.bfloat16, device=dev)
        out = prompt(q, k, v) if T == 0 else cached(q, k, v, T)
        assert (out == 2.0 ** e).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,Hq,Hkv,D", PROMPTS)
def test_neighbours_keep_their_bits_prompt(dev, n, Hq, Hkv, D, dt):
    """Infinities and NaN change the bits of nothing but the rows that see them, and of these, where only values are not
    finite, only those columns."""
    import torch
    say(f"neighbours, prompt {dt} n={n} Hq={Hq} D={D}")
    q, k, v = normals((n, Hq, D), dt, dev, 7), normals((n, Hkv, D), dt, dev, 8), normals((n, Hkv, D), dt, dev, 9)
    clean = prompt(q, k, v)
    for p, bad in ((n - 1, float("nan")), (n // 2 + 5, float("inf")), (97, float("-inf")), (0, float("nan"))):
        v2 = v.clone()
        v2[p, :, D - 3] = bad
        out = prompt(q, k, v2)
        rest = [d for d in range(D) if d != D - 3]
        assert torch.equal(out[:p], clean[:p]) and torch.equal(out[p:, :, rest], clean[p:, :, rest])
        assert not torch.isfinite(out[p:, :, D - 3]).any()
        k2 = k.clone()
        k2[p] = float("nan")
        out = prompt(q, k2, v2)
        assert torch.equal(out[:p], clean[:p]) and torch.isnan(out[p:]).all()


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,T,Hq,Hkv,D", [c for c in CACHES if c[1] > 1])
def test_neighbours_keep_their_bits_cache(dev, n, T, Hq, Hkv, D, dt):
    import torch
    say(f"neighbours, cache {dt} n={n} T={T} Hq={Hq} D={D}")
    q, k, v = normals((n, Hq, D), dt, dev, 10), normals((n, Hkv, D), dt, dev, 11), normals((n, Hkv, D), dt, dev, 12)
    tree = torch.tensor([[1 << t for t in range(T)]], dtype=torch.int64, device=dev)      # every draft on its own
    tree[0, 0] |= 1 << (T - 1)
    clean = cached(q, k, v, T, tree=tree)
    for t, bad in ((T - 1, float("inf")), (1, float("nan"))):
        v2, k2 = v.clone(), k.clone()
        v2[n - T + t, :, 2] = bad
        sees = [r for r in range(T) if r == t or (r == 0 and t == T - 1)]
        others = [r for r in range(T) if r not in sees]
        rest = [d for d in range(D) if d != 2]
        out = cached(q, k, v2, T, tree=tree)
        assert torch.equal(out[others], clean[others]) and torch.equal(out[:, :, rest], clean[:, :, rest])
        assert not torch.isfinite(out[sees][:, :, 2]).any()
        if bad == float("inf"):
            assert (out[sees][:, :, 2] == bad).all()
        k2[n - T + t] = float("nan")
        out = cached(q, k2, v2, T, tree=tree)
        assert torch.equal(out[others], clean[others]) and torch.isnan(out[sees]).all()


def test_alone_and_in_a_batch(dev):
    """Chunks depend on the number of sequences: a sequence alone agrees with itself in a batch within the bound."""
    import torch
    from attention_plain import check
    from forge_amd import ops
    B, n, T, Hq, Hkv, D, page = 5, 1500, 3, 8, 2, 128, 16
    pages = (n + page - 1) // page
    q = normals((B, T, Hq, D), "float16", dev, 20)
    kc, vc = normals((B * pages, page, Hkv, D), "float16", dev, 21), normals((B * pages, page, Hkv, D), "float16", dev, 22)
    table = torch.arange(B * pages, dtype=torch.int32, device=dev).view(B, pages)
    lens = torch.tensor([n - T, 700, 0, 64, 1111], dtype=torch.int32, device=dev)
    out = ops.cache_attention(q, kc, vc, table, lens)
    for b in range(B):
        alone = ops.cache_attention(q[b:b + 1], kc, vc, table[b:b + 1], lens[b:b + 1])
        m = int(lens[b]) + T
        seen = torch.arange(m, device=dev)[None] <= torch.arange(m - T, m, device=dev)[:, None]
        k, v = (c.view(B, -1, Hkv, D)[b, :m] for c in (kc, vc))
        for h in range(Hq):
            for got in (out[b, :, h], alone[0, :, h]):
                check(got, q[b, :, h], k[:, h // 4], v[:, h // 4], seen, D ** -0.5)


def test_longest_table(dev):
    """A table of 2^27 positions, the most that there may be."""
    import torch
    from forge_amd import ops
    page, n, D = 4096, 5000, 64
    q, k, v = normals((1, 1, 2, D), "float16", dev, 13), normals((2, page, 1, D), "float16", dev, 14), normals((2, page, 1, D), "float16", dev, 15)
    table = torch.full((1, (1 << 27) // page), -1, dtype=torch.int32, device=dev)
    table[0, :2] = torch.tensor([1, 0])
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    out = ops.cache_attention(q, k, v, table, lens)
    from attention_plain import check
    kk, vv = torch.cat([k[1], k[0]])[:n + 1, 0], torch.cat([v[1], v[0]])[:n + 1, 0]
    for h in range(2):
        check(out[0, :, h], q[0, :, h], kk, vv, torch.ones((1, n + 1), dtype=torch.bool, device=dev), D ** -0.5)


@pytest.mark.parametrize("keys", [30, 3000])
def test_many_sequences(dev, keys):
    """More sequences than a grid has rows: each its own query over one cache that they share."""
    import torch
    from attention_plain import check
    from forge_amd import ops
    B, D = 70001, 8
    page = 16 if keys < 100 else 4096
    q, k, v = normals((B, 1, 1, D), "float16", dev, 16), normals((2, page, 1, D), "float16", dev, 17), normals((2, page, 1, D), "float16", dev, 18)
    lens = keys - torch.arange(B, dtype=torch.int32, device=dev) % 3
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev).repeat(B, 1)
    out = ops.cache_attention(q, k, v, table, lens)
    for r in range(3):
        n = keys - r + 1
        rows = torch.arange(r, B, 3, device=dev)
        kk, vv = k.view(-1, D)[:n], v.view(-1, D)[:n]
        check(out[rows, 0, 0], q[rows, 0, 0], kk, vv, torch.ones((len(rows), n), dtype=torch.bool, device=dev), D ** -0.5)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 80, 128, 200])
def test_rows_past_the_end_are_zeros(dev, D, causal, dt):
    """Whatever the call before has left in LDS (NaN in every key and value here), the rows of a last tile that lie past the
    sequence count as zeros."""
    import torch
    say(f"rows past the end {dt} D={D} causal={causal}")
    for n, Hq, Hkv in ((300, 2, 1), (65, 64, 8), (1, 300, 300), (129, 200, 8), (700, 64, 8)):
        q, k, v = normals((n, Hq, D), dt, dev, n), normals((n, Hkv, D), dt, dev, n + 1), normals((n, Hkv, D), dt, dev, n + 2)
        nq, nk = normals((2048, 32, D), dt, dev, 1), torch.full((2048, 32, D), float("nan"), dtype=q.dtype, device=dev)
        want = prompt(q, k, v, causal=causal)
        assert torch.isfinite(want).all()
        for _ in range(3):
            left = prompt(nq, nk, nk, causal=causal)
            assert torch.equal(prompt(q, k, v, causal=causal), want)
        assert torch.isnan(left).all()
    for n, T, Hq, Hkv in ((100, 1, 4, 1), (900, 1, 8, 8), (333, 5, 16, 2), (1000, 61, 4, 1)):
        q, k, v = normals((n, Hq, D), dt, dev, n), normals((n, Hkv, D), dt, dev, n + 1), normals((n, Hkv, D), dt, dev, n + 2)
        want = cached(q, k, v, T)
        assert torch.isfinite(want).all()
        for _ in range(3):
            prompt(nq, nk, nk, causal=causal)
            assert torch.equal(cached(q, k, v, T), want)


# ---- compiled calls ------------------------------------------------------------------------------

def test_both_call_paths_agree(dev, monkeypatch):
    """The compiled call and the checks with the foreign call behind them hand over the same arguments."""
    import torch
    from forge_amd import ops
    calls = []

    def both(name, f):
        fast = f()
        with monkeypatch.context() as m:
            m.setattr(ops, "_fast", lambda called, *a: calls.append(called))
            slow = f()
        for a, b in zip(fast, slow):
            assert torch.equal(a, b), name

    x, q4, s, w = int4_case(7, 384, 50, "bfloat16", dev, 1)
    bias = torch.randn((50,), device=dev).to(torch.bfloat16)
    both("int4_linear", lambda: [ops.int4_linear(x, w, s, bias)])
    T, Hq, Hkv, D = 40, 6, 2, 80
    qkv = normals((T, Hq + 2 * Hkv, D), "float16", dev, 2)
    q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
    cos, sin = torch.rand((64, 24), device=dev), torch.rand((64, 24), device=dev)
    pos = torch.randint(0, 64, (T,), device=dev, dtype=torch.int32)
    slots = torch.randperm(48, device=dev)[:T].to(torch.int32)
    nw = torch.rand((D,), device=dev).half()
    for inter in (False, True):
        both("qk_norm_rope", lambda: ops.qk_norm_rope(q, k, nw, None, cos, sin, pos, eps=1e-5, interleaved=inter))

        def into_cache():
            kc, vc = (torch.zeros((3, 16, Hkv, D), dtype=torch.float16, device=dev) for _ in range(2))
            ko = torch.empty((T, Hkv, D), dtype=torch.float16, device=dev)
            return ops.qk_norm_rope_cache(q, k, v, None, nw, cos, sin, pos, kc, vc, slots, interleaved=inter, k_out=ko), ko, kc, vc
        both("qk_norm_rope_cache", into_cache)
    cu = torch.tensor([0, 13, 40], dtype=torch.int32, device=dev)
    for causal in (False, True):
        both("prompt_attention", lambda: [ops.prompt_attention(q, k, v, cu, 0.3, causal)])
    B, T = 2, 3
    q = normals((B, T, Hq, D), "float16", dev, 3)
    kc, vc = normals((5, 16, Hkv, D), "float16", dev, 4), normals((5, 16, Hkv, D), "float16", dev, 5)
    table = torch.tensor([[4, 0, 2], [1, 3, 0]], dtype=torch.int32, device=dev)
    lens = torch.tensor([40, 17], dtype=torch.int32, device=dev)
    tree = torch.tensor([[1, 3, 5], [1, 2, 7]], device=dev)
    ws = torch.empty((max(16, ops.cache_attention_workspace_size(B, T, Hq, Hkv, D, 48)),), dtype=torch.uint8, device=dev)
    for tr in (None, tree):
        both("cache_attention", lambda: [ops.cache_attention(q, kc, vc, table, lens, tr, workspace=ws, out=torch.empty_like(q))])
    assert set(calls) == {"int4_linear", "qk_norm_rope", "prompt_attention", "cache_attention"}
