"""The decoder-attention operators whose speed is measured: linear layers with 4-bit weights, per-head norm
and rotation of queries and keys (with the write into a paged cache), attention over packed prompts,
and attention over a paged cache for single tokens and for trees of drafted tokens.

A case is a dict of plain values: "kind" and the sizes. listed() holds the fixed ones, draw() gives
further cases of the same ranges. run() makes the framework's calls where `own` is true, and
computes the same results from elementary torch operations in 32 bits where it is false.
"""
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # One token through a square projection: the smallest call, bound by latency.
        {"name": "int4 1x4096x4096", "kind": "int4", "M": 1, "K": 4096, "N": 4096, "G": 128, "bias": False,
         "dtype": "float16"},
        # A few sequences decoding together; fine scales, a K that is no multiple of 128, an odd number of rows.
        {"name": "int4 5x2880x2881 bf16", "kind": "int4", "M": 5, "K": 2880, "N": 2881, "G": 32, "bias": True,
         "dtype": "bfloat16"},
        # 64 drafted tokens verified at once through the widest layer: the most tokens the operator is meant for.
        {"name": "int4 64x8192x11008", "kind": "int4", "M": 64, "K": 8192, "N": 11008, "G": 128, "bias": True,
         "dtype": "float16"},
        # A decode step of 8 sequences: latency; K and V go into the cache.
        {"name": "rope 8 tokens into cache", "kind": "rope", "T": 8, "Hq": 32, "Hkv": 8, "D": 128, "R": 128,
         "interleaved": False, "cache": True, "dtype": "float16"},
        # An odd prompt of a small model that rotates half of each head in neighbouring pairs.
        {"name": "rope 1501 tokens bf16", "kind": "rope", "T": 1501, "Hq": 16, "Hkv": 16, "D": 64, "R": 32,
         "interleaved": True, "cache": False, "dtype": "bfloat16"},
        # A long prompt of a wide model on its way into the cache: bandwidth.
        {"name": "rope 16384 tokens into cache", "kind": "rope", "T": 16384, "Hq": 64, "Hkv": 8, "D": 128, "R": 128,
         "interleaved": False, "cache": True, "dtype": "float16"},
        # Short prompts of different lengths packed together, one of a single token, one empty.
        {"name": "prompt packed short bf16", "kind": "prompt", "lens": "1,37,200,0,511,64,130", "Hq": 16, "Hkv": 16,
         "D": 64, "causal": True, "dtype": "bfloat16"},
        # One prompt of ordinary length, grouped heads.
        {"name": "prompt 4096", "kind": "prompt", "lens": "4096", "Hq": 32, "Hkv": 8, "D": 128, "causal": True,
         "dtype": "float16"},
        # A batch of long prompts packed without padding: the largest call, bound by the matrix units.
        {"name": "prompt packed 16384", "kind": "prompt", "lens": "9001,5120,2263", "Hq": 32, "Hkv": 8, "D": 128,
         "causal": True, "dtype": "bfloat16"},
        # One sequence, one token: the latency of decode.
        {"name": "cache 1x1 over 1000", "kind": "cache", "lens": "1000", "T": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "dtype": "float16"},
        # Trees of 61 drafted tokens for a few sequences (one not begun), groups of eight heads.
        {"name": "cache 4x61 tree bf16", "kind": "cache", "lens": "3001,17,0,2048", "T": 61, "Hq": 16, "Hkv": 2, "D": 64,
         "page": 32, "dtype": "bfloat16"},
        # A serving batch of ragged lengths, 16 drafts each: bandwidth of the cache.
        {"name": "cache 16x16 long", "kind": "cache",
         "lens": "32768,30011,28000,517,16384,8191,24000,12345,4096,20480,31000,65,2000,9999,27001,15000", "T": 16,
         "Hq": 32, "Hkv": 8, "D": 128, "page": 64, "dtype": "float16"},
    ]


def _log_int(rng, lo, hi):
    """Uniform over the logarithm; whole multiples of 1024 are left to the listed cases."""
    n = max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return n if n % 1024 else n - 1


def draw(rng):
    kind = rng.choice(["int4", "rope", "prompt", "cache"])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "int4":
        G = rng.choice([32, 64, 128])
        while True:
            c = {"kind": kind, "M": _log_int(rng, 1, 64), "K": G * (_log_int(rng, 1024 // G, 11008 // G) | 1),
                 "N": _log_int(rng, 257, 28000), "G": G, "bias": rng.random() < 0.5, "dtype": dtype}
            if c["K"] * c["N"] <= 8192 * 11008:
                return c
    if kind == "rope":
        D = rng.choice([64, 80, 96, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        R = rng.choice([D, D // 2 // 16 * 16])
        while True:
            c = {"kind": kind, "T": _log_int(rng, 1, 16384), "Hq": Hkv * rng.choice([1, 2, 3, 4, 7, 8]), "Hkv": Hkv,
                 "D": D, "R": R, "interleaved": rng.random() < 0.4, "cache": rng.random() < 0.6, "dtype": dtype}
            if c["T"] * (c["Hq"] + 2 * Hkv) * D <= 16384 * 80 * 128:
                return c
    if kind == "prompt":
        D = rng.choice([64, 64, 80, 128, 128, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 5, 8])
        n = _log_int(rng, 1, 12)
        while True:
            lens = [_log_int(rng, 1, 9001) for _ in range(n)]
            c = {"kind": kind, "lens": ",".join(map(str, lens)), "Hq": Hq, "Hkv": Hkv, "D": D,
                 "causal": rng.random() < 0.85, "dtype": dtype}
            if work(c)["flops"] <= work(_named("prompt packed 16384"))["flops"]:
                return c
    D = rng.choice([64, 80, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    B = _log_int(rng, 1, 32)
    while True:
        lens = [rng.choice([0, 1, 2, 3, 4, 5, 6, 7]) and _log_int(rng, 1, 32768) for _ in range(B)]
        c = {"kind": kind, "lens": ",".join(map(str, lens)), "T": rng.choice([1, 1, _log_int(rng, 2, 64)]),
             "Hq": Hkv * rng.choice([1, 2, 4, 7, 8]), "Hkv": Hkv, "D": D, "page": rng.choice([16, 32, 64, 128]),
             "dtype": dtype}
        most = work(_named("cache 16x16 long"))
        if work(c)["bytes"] <= most["bytes"] and work(c)["flops"] <= most["flops"]:
            return c


def _named(name):
    return next(c for c in listed() if c["name"] == name)


def _lens(c):
    return [int(n) for n in c["lens"].split(",")]


def _dtype(c):
    return getattr(torch, c["dtype"])


# ---- inputs -----------------------------------------------------------------------------------

def _pack_int4(q):
    """(N, K) integers in -8..7 -> (N, ceil(K / 128) * 64) bytes: rows of 128-value blocks, each a 4 x 4
    transpose of its 32-bit words (word 4 g + j holds values 32 j + 8 g to + 7), of whose eight
    values (+ 8) the even ones lie at bits 0, 4, 8, 12 and the odd ones 16 bits further up."""
    N, K = q.shape
    blocks = (K + 127) // 128
    full = torch.zeros((N, blocks * 128), dtype=torch.int64, device=q.device)
    full[:, :K] = q
    u = (full + 8).view(N, blocks, 4, 4, 4, 2)                        # j, g, pair, even / odd
    shift = torch.tensor([[4 * i, 4 * i + 16] for i in range(4)], device=q.device)
    words = (u << shift).sum((-1, -2)).transpose(2, 3).reshape(N, blocks * 16)   # g, j
    out = torch.stack([(words >> (8 * b)) & 255 for b in range(4)], dim=-1)
    return out.to(torch.uint8).reshape(N, blocks * 64)


def _unpack_int4(w, K):
    N = w.shape[0]
    b = w.view(N, -1, 4, 4, 4).transpose(2, 3)                        # block, j, g, byte of the word
    lo, hi = b & 15, b >> 4                                          # nibbles 2 byte and 2 byte + 1
    nib = torch.stack([lo, hi], dim=-1).reshape(N, -1, 4, 4, 8)       # nibble position in the word
    v = torch.stack([nib[..., :4], nib[..., 4:]], dim=-1)             # pair, even / odd
    return v.reshape(N, -1)[:, :K].to(torch.int32) - 8


def prepare(case, seed):
    c, dt = case, _dtype(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = random.Random(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s = {"case": c}
    if c["kind"] == "int4":
        M, K, N, G = c["M"], c["K"], c["N"], c["G"]
        q = (randn(N, K) * 2.5).round().clamp(-8, 7).to(torch.int8)
        s["w"] = _pack_int4(q)
        s["ws"] = (torch.rand((N, K // G), generator=g, device=DEV) * 6e-3 + 2e-3).half()
        x = randn(M, K)
        x[:, ::509] *= 8.0                                           # outlier channels
        s["x"] = x.to(dt)
        s["bias"] = (randn(N) * 0.1).to(dt) if c["bias"] else None
        s["out"] = torch.empty((M, N), dtype=dt, device=DEV)
    elif c["kind"] == "rope":
        T, Hq, Hkv, D, R = c["T"], c["Hq"], c["Hkv"], c["D"], c["R"]
        qkv = (randn(T, Hq + 2 * Hkv, D) * 1.5).to(dt)               # the projection's output
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        s["qw"] = (torch.rand((D,), generator=g, device=DEV) + 0.5).to(dt)
        s["kw"] = (torch.rand((D,), generator=g, device=DEV) + 0.5).to(dt)
        P = T + 1000
        angle = torch.arange(P, device=DEV)[:, None] * 10000.0 ** (-torch.arange(R // 2, device=DEV) * (2.0 / R))
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        s["pos"] = (torch.arange(T, device=DEV) + rng.randrange(1000)).to(torch.int32)
        s["q_out"] = torch.empty((T, Hq, D), dtype=dt, device=DEV)
        if c["cache"]:
            page, pages = 16, (T + 15) // 16 + 3
            s["kc"] = randn(pages, page, Hkv, D).to(dt)
            s["vc"] = randn(pages, page, Hkv, D).to(dt)
            order = torch.randperm(pages, generator=g, device=DEV)
            at = torch.arange(T, device=DEV)
            s["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        else:
            s["k_out"] = torch.empty((T, Hkv, D), dtype=dt, device=DEV)
    elif c["kind"] == "prompt":
        lens, Hq, Hkv, D = _lens(c), c["Hq"], c["Hkv"], c["D"]
        T = sum(lens)
        # queries and keys are normed heads, values are still where the projection wrote them
        w = torch.rand((D,), generator=g, device=DEV) + 0.5
        s["q"], s["k"] = (randn(T, Hq, D) * w).to(dt), (randn(T, Hkv, D) * w).to(dt)
        s["v"] = randn(T, Hq + 2 * Hkv, D).to(dt)[:, Hq + Hkv:]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["out"] = torch.empty((T, Hq, D), dtype=dt, device=DEV)
    else:
        lens, T, Hq, Hkv, D, page = _lens(c), c["T"], c["Hq"], c["Hkv"], c["D"], c["page"]
        B = len(lens)
        need = [(n + T + page - 1) // page for n in lens]
        pages = sum(need) + 5
        w = torch.rand((D,), generator=g, device=DEV) + 0.5
        s["q"] = (randn(B, T, Hq, D) * w).to(dt)
        s["kc"] = torch.empty((pages, page, Hkv, D), dtype=dt, device=DEV)
        s["vc"] = torch.empty((pages, page, Hkv, D), dtype=dt, device=DEV)
        for i in range(0, pages, 256):
            n = min(256, pages - i)
            s["kc"][i:i + n] = (randn(n, page, Hkv, D) * w).to(dt)
            s["vc"][i:i + n] = randn(n, page, Hkv, D).to(dt)
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        s["table"] = torch.zeros((B, max(need)), dtype=torch.int32, device=DEV)
        at = 0
        for b in range(B):
            s["table"][b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["tree"] = None
        if T > 1:
            rows = []
            for b in range(B):
                bits = []
                for t in range(T):                                    # each draft hangs on an earlier one or on the cache
                    parent = rng.randrange(-1, t) if t else -1
                    m = (1 << t) | (bits[parent] if parent >= 0 else 0)
                    bits.append(m)
                rows.append([m - (1 << 64) if m >> 63 else m for m in bits])
            s["tree"] = torch.tensor(rows, dtype=torch.int64, device=DEV)
        s["out"] = torch.empty((B, T, Hq, D), dtype=dt, device=DEV)
        if own:
            from forge_amd import ops
            size = ops.cache_attention_workspace_size(B, T, Hq, Hkv, D, max(need) * page)
            s["workspace"] = torch.empty((size,), dtype=torch.uint8, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from forge_amd import ops
    c = s["case"]
    if c["kind"] == "int4":
        return ops.int4_linear(s["x"], s["w"], s["ws"], s["bias"], out=s["out"])
    if c["kind"] == "rope":
        if not c["cache"]:
            return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], eps=EPS,
                                    interleaved=c["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
        q = ops.qk_norm_rope_cache(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], s["kc"],
                                   s["vc"], s["slots"], eps=EPS, interleaved=c["interleaved"], q_out=s["q_out"])
        return q, s["kc"], s["vc"]
    if c["kind"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"], out=s["out"])
    return ops.cache_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], tree=s["tree"],
                               workspace=s["workspace"], out=s["out"])


def _norm_rope_plain(x, w, cos, sin, interleaved):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    h = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([rot, x[..., 2 * h:]], dim=-1)


def _softmax_rows(scores, seen):
    """Row softmax over the seen entries; rows that see nothing are zeros."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _run_plain(s):
    c, dt = s["case"], _dtype(s["case"])
    if c["kind"] == "int4":
        w = _unpack_int4(s["w"], c["K"]).float() * s["ws"].float().repeat_interleave(c["G"], dim=1)
        y = s["x"].float() @ w.T
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(dt)
    if c["kind"] == "rope":
        pos = s["pos"].long()
        cos, sin = s["cos"][pos], s["sin"][pos]
        q = _norm_rope_plain(s["q"], s["qw"], cos, sin, c["interleaved"]).to(dt)
        k = _norm_rope_plain(s["k"], s["kw"], cos, sin, c["interleaved"]).to(dt)
        if not c["cache"]:
            return q, k
        slots = s["slots"].long()
        s["kc"].view(-1, c["Hkv"], c["D"])[slots] = k
        s["vc"].view(-1, c["Hkv"], c["D"])[slots] = s["v"]
        return q, s["kc"], s["vc"]
    scale = 1.0 / math.sqrt(c["D"])
    group = c["Hq"] // c["Hkv"]
    if c["kind"] == "prompt":
        out, at = torch.empty_like(s["out"]), 0
        for L in _lens(c):
            if L == 0:
                continue
            i = torch.arange(L, device=DEV)
            seen = i[None, :] <= i[:, None] if c["causal"] else torch.ones((L, L), dtype=torch.bool, device=DEV)
            for h in range(c["Hkv"]):
                k, v = s["k"][at:at + L, h].float(), s["v"][at:at + L, h].float()
                for hq in range(h * group, (h + 1) * group):
                    scores = (s["q"][at:at + L, hq].float() @ k.T.contiguous()) * scale
                    out[at:at + L, hq] = (_softmax_rows(scores, seen) @ v).to(dt)
            at += L
        return out
    T, page = c["T"], c["page"]
    out = torch.empty_like(s["out"])
    j = torch.arange(T, device=DEV)
    for b, L in enumerate(_lens(c)):
        pages = s["table"][b, :(L + T + page - 1) // page].long()
        k = s["kc"][pages].flatten(0, 1)[:L + T].float().permute(1, 2, 0).contiguous()      # head, dim, key
        v = s["vc"][pages].flatten(0, 1)[:L + T].float().permute(1, 0, 2).contiguous()      # head, key, dim
        q = s["q"][b].float().view(T, c["Hkv"], group, c["D"]).permute(1, 0, 2, 3).reshape(c["Hkv"], T * group, c["D"])
        if s["tree"] is None:
            drafts = j[None, :] <= j[:, None]
        else:
            drafts = ((s["tree"][b][:, None] >> j) & 1) == 1
        seen = torch.cat([torch.ones((T, L), dtype=torch.bool, device=DEV), drafts], dim=1).repeat_interleave(group, 0)
        o = _softmax_rows(torch.matmul(q, k) * scale, seen) @ v
        out[b] = o.view(c["Hkv"], T, group, c["D"]).permute(1, 0, 2, 3).reshape(T, c["Hq"], c["D"]).to(dt)
    return out


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; a multiply-add is two operations."""
    c = case
    if c["kind"] == "int4":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": 2 * M * K + N * K // 2 + 2 * N * K // c["G"] + 2 * M * N + (2 * N if c["bias"] else 0),
                "flops": 2 * M * N * K}
    if c["kind"] == "rope":
        heads = c["Hq"] + (2 if c["cache"] else 1) * c["Hkv"]
        return {"bytes": c["T"] * (4 * heads * c["D"] + 4 * c["R"] + (8 if c["cache"] else 4)) + 4 * c["D"],
                "flops": c["T"] * (c["Hq"] + c["Hkv"]) * (4 * c["D"] + 3 * c["R"])}
    if c["kind"] == "prompt":
        lens = _lens(c)
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (4 * c["Hq"] + 4 * c["Hkv"]) * c["D"] + 4 * (len(lens) + 1),
                "flops": 4 * c["D"] * c["Hq"] * pairs}
    lens, T = _lens(c), c["T"]
    keys = sum(n + T for n in lens)
    return {"bytes": 4 * keys * c["Hkv"] * c["D"] + 4 * len(lens) * T * c["Hq"] * c["D"] + 8 * len(lens) * T
            + 4 * len(lens) + 4 * sum((n + T + c["page"] - 1) // c["page"] for n in lens),
            "flops": 4 * c["D"] * c["Hq"] * T * keys}


# ---- the same results in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    D = c.get("D", 0)
    if c["kind"] == "int4":
        words = s["w"].to(torch.int64)
        N = words.shape[0]
        y = torch.zeros((c["M"], N), dtype=torch.float64, device=DEV)
        for k0 in range(0, c["K"], 32):                              # one 32-deep slice: word column j of its block
            block, j = k0 // 128, k0 // 32 % 4
            part = torch.empty((N, 32), dtype=torch.float64, device=DEV)
            for k in range(32):
                word, e = 4 * (k // 8) + j, k % 8
                bit = 4 * (e // 2) + 16 * (e % 2)
                byte = words[:, block * 64 + 4 * word + bit // 8]
                part[:, k] = ((byte >> (bit % 8)) & 15).double() - 8.0
            y += (s["x"][:, k0:k0 + 32].double() @ part.T) * s["ws"][:, k0 // c["G"]].double()
        return y + s["bias"].double() if s["bias"] is not None else y
    if c["kind"] == "rope":
        def rotate(x, w):
            x = x.double()
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
            h = c["R"] // 2
            z = torch.complex(s["cos"][s["pos"].long()].double(), s["sin"][s["pos"].long()].double())[:, None]
            first = torch.arange(h, device=DEV) * (2 if c["interleaved"] else 1)
            second = first + (1 if c["interleaved"] else h)
            turned = torch.complex(x[..., first], x[..., second]) * z
            y = x.clone()
            y[..., first], y[..., second] = turned.real, turned.imag
            return y
        q, k = rotate(s["q"], s["qw"]), rotate(s["k"], s["kw"])
        if not c["cache"]:
            return q, k
        kc, vc = s["kc"].double(), s["vc"].double()
        page = kc.shape[1]
        kc[s["slots"].long() // page, s["slots"].long() % page] = k
        vc[s["slots"].long() // page, s["slots"].long() % page] = s["v"].double()
        return q, kc, vc
    group = c["Hq"] // c["Hkv"]
    if c["kind"] == "prompt":
        out, at = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV), 0
        for L in _lens(c):
            for h in range(c["Hq"]):
                k, v = s["k"][at:at + L, h // group].double(), s["v"][at:at + L, h // group].double()
                for i in range(0, L, 2048):
                    n = min(i + 2048, L)
                    e = n if c["causal"] else L
                    z = s["q"][at + i:at + n, h].double() @ k[:e].T.contiguous() / math.sqrt(D)
                    if c["causal"]:
                        z += torch.full((n - i, e), -math.inf, dtype=torch.float64, device=DEV).triu(i + 1)
                    out[at + i:at + n, h] = torch.softmax(z, -1) @ v[:e]
            at += L
        return out
    T, page = c["T"], c["page"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for b, L in enumerate(_lens(c)):
        at = torch.arange(L + T, device=DEV)
        rows = s["table"][b].long()[at // page] * page + at % page
        if T == 1:
            hidden = torch.zeros((1, L + 1), dtype=torch.float64, device=DEV)
        else:
            bits = [[0.0 if (m >> t) & 1 else -math.inf for t in range(T)] for m in s["tree"][b].tolist()]
            hidden = torch.zeros((T, L + T), dtype=torch.float64, device=DEV)
            hidden[:, L:] = torch.tensor(bits, dtype=torch.float64, device=DEV)
        for h in range(c["Hkv"]):
            k = s["kc"].view(-1, c["Hkv"], D)[rows, h].double()
            v = s["vc"].view(-1, c["Hkv"], D)[rows, h].double()
            for hq in range(h * group, (h + 1) * group):
                z = s["q"][b, :, hq].double() @ k.T.contiguous() / math.sqrt(D) + hidden
                out[b, :, hq] = torch.softmax(z, -1) @ v
    return out
