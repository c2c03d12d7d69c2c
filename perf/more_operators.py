"""The operators of several continuations over a 4-bit cache whose speed is measured: keys and values into and out
of a paged cache of 4 bits a value, attention over that cache, the selection of a beam search's next tokens, and the pages of
its rows after it (shared, copied, taken anew).

A case is a dict of plain values: "kind" and the sizes. listed() holds the fixed ones, draw() gives
further cases of the same ranges. run() makes the framework's calls where `own` is true, and
computes the same results from elementary torch operations where it is false.

The cache: uint8 (pages, KV heads, page size, 32 U + 8) with U = 2, 3, 4, 6 or 8, the smallest with D <= 32 U. The
bytes of a page's head are page size rows of keys (4 U words of 32 bits, word n the values 8 n to 8 n + 7, of these value 2 i at bits 4 i
and value 2 i + 1 at bits 16 + 4 i), then the rows of values, the same words of four positions side by side
(position / 4, word, position % 4), then per position four 16-bit numbers: step and lowest value of its key, and of its value.
"""
import math
import random

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # A decode step of 8 sequences: their keys and values into the cache, latency.
        {"name": "store 8 tokens", "kind": "store", "T": 8, "Hq": 32, "Hkv": 8, "D": 128, "page": 16, "dtype": "float16"},
        # An odd prompt of a small model with heads that fill no whole row.
        {"name": "store 1501 tokens bf16", "kind": "store", "T": 1501, "Hq": 12, "Hkv": 4, "D": 80, "page": 32,
         "dtype": "bfloat16"},
        # A long prompt on its way into the cache: bandwidth.
        {"name": "store 16384 tokens", "kind": "store", "T": 16384, "Hq": 64, "Hkv": 8, "D": 128, "page": 64,
         "dtype": "float16"},
        # One sequence, one token: the latency of decode.
        {"name": "attend 1x1 over 1000", "kind": "attend", "lens": "1000", "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "float16"},
        # Trees of 29 drafts for a few sequences (one not begun), groups of seven heads.
        {"name": "attend 4x29 tree bf16", "kind": "attend", "lens": "3001,17,0,2048", "T": 29, "Hq": 14, "Hkv": 2, "D": 64,
         "page": 32, "dtype": "bfloat16"},
        # A serving batch of ragged lengths, one token each: bandwidth of the cache.
        {"name": "attend 16x1 long", "kind": "attend",
         "lens": "32768,30011,28000,517,16384,8191,24000,12345,4096,20480,31000,65,2000,9999,27001,15000", "T": 1,
         "Hq": 32, "Hkv": 8, "D": 128, "page": 64, "dtype": "float16"},
        # A few long sequences with trees of 16 drafts: the most operations.
        {"name": "attend 6x16 long bf16", "kind": "attend", "lens": "32768,28001,16384,9999,31000,517", "T": 16, "Hq": 32,
         "Hkv": 4, "D": 128, "page": 64, "dtype": "bfloat16"},
        # Four beams of one request: latency.
        {"name": "beams 1x4 of 32000", "kind": "beams", "B": 1, "W": 4, "V": 32000, "count": 8, "ended": False,
         "dtype": "float16"},
        # A vocabulary of odd size, some beams that have ended.
        {"name": "beams 16x5 of 50257 bf16", "kind": "beams", "B": 16, "W": 5, "V": 50257, "count": 5, "ended": True,
         "dtype": "bfloat16"},
        # Many requests, a large vocabulary, 32-bit logits: bandwidth.
        {"name": "beams 32x8 of 131072", "kind": "beams", "B": 32, "W": 8, "V": 131072, "count": 16, "ended": True,
         "dtype": "float32"},
        # The rows of one request after a selection, caches of two layers: latency.
        {"name": "fork 1x4", "kind": "fork", "B": 1, "W": 4, "prompt": 300, "most": 100, "width": 40, "page": 16, "Hkv": 8,
         "D": 128, "tensors": 4, "dtype": "float16"},
        # The rows of many requests: bandwidth of the copied pages.
        {"name": "fork 64x8", "kind": "fork", "B": 64, "W": 8, "prompt": 320, "most": 60, "width": 128, "page": 16, "Hkv": 4,
         "D": 128, "tensors": 8, "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    """Uniform over the logarithm; whole multiples of 1024 are left to the listed cases."""
    n = max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return n if n % 1024 else n - 1


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "beams", "fork"])
    dtype = rng.choice(["float16", "bfloat16"])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    while True:
        if kind == "store":
            c = {"kind": kind, "T": _log_int(rng, 1, 16384), "Hq": Hkv * rng.choice([1, 2, 4, 7, 8]), "Hkv": Hkv, "D": D,
                 "page": page, "dtype": dtype}
            if c["T"] * Hkv * D <= 16384 * 8 * 128:
                return c
        elif kind == "attend":
            lens = [rng.choice([0, 1, 2, 3, 4, 5, 6, 7]) and _log_int(rng, 1, 32768) for _ in range(_log_int(rng, 1, 32))]
            c = {"kind": kind, "lens": ",".join(map(str, lens)), "T": rng.choice([1, 1, 1, _log_int(rng, 2, 64)]),
                 "Hq": Hkv * rng.choice([1, 2, 4, 7, 8]), "Hkv": Hkv, "D": D, "page": page, "dtype": dtype}
            if (work(c)["bytes"] <= work(_named("attend 16x1 long"))["bytes"]
                    and work(c)["flops"] <= work(_named("attend 6x16 long bf16"))["flops"]):
                return c
        elif kind == "beams":
            W = _log_int(rng, 1, 16)
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "W": W, "V": _log_int(rng, 500, 200000),
                 "count": rng.choice([W, 2 * W, _log_int(rng, 1, 64)]), "ended": rng.random() < 0.4,
                 "dtype": rng.choice(["float16", "bfloat16", "float32"])}
            if c["B"] * W * c["V"] <= 32 * 8 * 131072:
                return c
        else:
            most = _log_int(rng, 1, 200)
            prompt = _log_int(rng, 1, 1500)
            c = {"kind": kind, "B": _log_int(rng, 1, 64), "W": _log_int(rng, 2, 16), "prompt": prompt, "most": most,
                 "width": (prompt + most) // page + rng.choice([1, 2, 9, 40]), "page": page, "Hkv": Hkv, "D": D,
                 "tensors": rng.choice([1, 2, 4, 6, 8]), "dtype": dtype}
            size = c["tensors"] * page * Hkv * D
            if _pages(c) * size <= 4200 * 8 * 16 * 4 * 128 and c["B"] * c["W"] * size <= 512 * 8 * 16 * 4 * 128:
                return c


def _named(name):
    return next(c for c in listed() if c["name"] == name)


def _lens(c):
    return [int(n) for n in c["lens"].split(",")]


def _dtype(c):
    return getattr(torch, c["dtype"])


def _words(D):
    """Words of 8 values that a head takes."""
    return 4 * next(u for u in (2, 3, 4, 6, 8) if D <= 32 * u)


def _pages(c):
    """Pages that a fork case's pool has."""
    return c["B"] * (c["prompt"] // c["page"] + c["W"] * (c["most"] // c["page"] + 3)) + 5


# ---- the cache's layout -------------------------------------------------------------------------

_SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]


def _pack(n, D):
    """(.., D) integers 0 to 15 -> (.., words, 4) bytes."""
    W = _words(D)
    full = torch.zeros(n.shape[:-1] + (8 * W,), dtype=torch.int64, device=n.device)
    full[..., :D] = n
    words = (full.view(*n.shape[:-1], W, 8) << torch.tensor(_SHIFTS, device=n.device)).sum(-1)
    return torch.stack([(words >> (8 * b)) & 255 for b in range(4)], dim=-1).to(torch.uint8)


def _unpack(b, D):
    """(.., words, 4) bytes -> (.., D) integers."""
    nib = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)            # nibble positions 0 to 7 of each word
    n = torch.stack([nib[..., :4], nib[..., 4:]], dim=-1).flatten(-2)   # 0, 4, 1, 5, ..
    return n.flatten(-2)[..., :D]


def _parts(cache, page, D):
    """Views of a cache: key bytes (pages, heads, page, words, 4), value bytes (pages, heads, page / 4, words, 4, 4)
    and numbers (pages, heads, page, 4, 2)."""
    W = _words(D)
    flat = cache.flatten(2)
    shape = flat.shape[:2]
    return (flat[..., :page * 4 * W].view(*shape, page, W, 4),
            flat[..., page * 4 * W:page * 8 * W].view(*shape, page // 4, W, 4, 4),
            flat[..., page * 8 * W:].view(*shape, page, 4, 2))


def _toward_zero(x, dt):
    """x >= 0 in 32 bits, rounded toward zero to dt."""
    y = x.to(dt)
    return torch.where(y.float() > x, (y.view(torch.int16) - 1).view(dt), y)


def _quantize(x):
    """(.., D) of 16 bits -> integers, step, lowest value; heads that are not finite get NaN for both."""
    f = x.float()
    low, top = f.amin(-1), f.amax(-1)
    part = torch.full_like(low, 15.0)                               # (a tensor: a number would be multiplied by its reciprocal)
    step = _toward_zero(top / part - low / part, x.dtype)
    s = step.float()[..., None]
    n = ((f * 0.5 - low[..., None] * 0.5) / (s * 0.5)).round()
    n = torch.where(s > 0.0, n, 0.0).clamp(0.0, 15.0)
    odd = ~torch.isfinite(f).all(-1)
    nan = torch.full_like(step, float("nan"))
    return (torch.where(odd[..., None], 0.0, n).to(torch.int64), torch.where(odd, nan, step),
            torch.where(odd, nan, low.to(x.dtype)))


# ---- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    c, dt = case, None if case["kind"] == "beams" else _dtype(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = random.Random(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s = {"case": c}
    if c["kind"] == "store":
        T, Hkv, D, page = c["T"], c["Hkv"], c["D"], c["page"]
        x = randn(T, c["Hq"] + 2 * Hkv, D) * 1.5                        # the projection's output
        x[:, :, ::37] *= 4.0                                           # outlier channels
        x = x.to(dt)
        s["k"], s["v"] = x[:, c["Hq"]:c["Hq"] + Hkv], x[:, c["Hq"] + Hkv:]
        pages = (T + page - 1) // page + 3
        s["cache"] = torch.zeros((pages, Hkv, page, 8 * _words(D) + 8), dtype=torch.uint8, device=DEV)
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(T, device=DEV)
        s["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        s["k_out"] = torch.empty((T, Hkv, D), dtype=dt, device=DEV)
        s["v_out"] = torch.empty((T, Hkv, D), dtype=dt, device=DEV)
    elif c["kind"] == "attend":
        lens, T, Hq, Hkv, D, page = _lens(c), c["T"], c["Hq"], c["Hkv"], c["D"], c["page"]
        B = len(lens)
        need = [(n + T + page - 1) // page for n in lens]
        pages = sum(need) + 5
        s["q"] = (randn(B, T, Hq, D) * (torch.rand((D,), generator=g, device=DEV) + 0.5)).to(dt)
        s["cache"] = torch.zeros((pages, Hkv, page, 8 * _words(D) + 8), dtype=torch.uint8, device=DEV)
        kb, vb, numbers = _parts(s["cache"], page, D)
        for i in range(0, pages, 256):
            n = min(256, pages - i)
            # about what the values of a head are after their quantization
            kb[i:i + n] = _pack((randn(n, Hkv, page, D) * 2.8 + 7.5).round().clamp(0, 15).to(torch.int64), D)
            v = _pack((randn(n, Hkv, page, D) * 2.8 + 7.5).round().clamp(0, 15).to(torch.int64), D)
            vb[i:i + n] = v.view(n, Hkv, page // 4, 4, -1, 4).transpose(3, 4)
            step = torch.rand((n, Hkv, page, 2), generator=g, device=DEV) * 0.2 + 0.25
            low = -step * (6.5 + 2.0 * torch.rand((n, Hkv, page, 2), generator=g, device=DEV))
            numbers[i:i + n] = torch.stack([step, low], -1).to(dt).view(torch.uint8).view(n, Hkv, page, 4, 2)
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
                    bits.append((1 << t) | (bits[parent] if parent >= 0 else 0))
                rows.append([m - (1 << 64) if m >> 63 else m for m in bits])
            s["tree"] = torch.tensor(rows, dtype=torch.int64, device=DEV)
        s["out"] = torch.empty((B, T, Hq, D), dtype=dt, device=DEV)
        if own:
            from forge_amd import ops
            size = ops.cache4_attention_workspace_size(B, T, Hq, Hkv, D, max(need) * page)
            s["workspace"] = torch.empty((size,), dtype=torch.uint8, device=DEV)
    elif c["kind"] == "beams":
        B, W, V, n = c["B"], c["W"], c["V"], c["count"]
        x = randn(B, W, V) * 2.5
        x[:, :, :16] += 6.0                                            # a few likely tokens
        x[:, :, V // 3:V // 3 + V // 50] = float("-inf")               # banned ones
        s["logits"] = x.to(_dtype(c))
        s["scores"] = -(torch.rand((B, W), generator=g, device=DEV) * 3.0).cumsum(-1)
        s["ended"], s["end"] = None, V - 1
        if c["ended"]:
            s["ended"] = torch.rand((B, W), generator=g, device=DEV) < 0.3
        s["out"] = (torch.empty((B, n), dtype=torch.float32, device=DEV),
                    torch.empty((B, n), dtype=torch.int32, device=DEV), torch.empty((B, n), dtype=torch.int32, device=DEV))
        if own:
            from forge_amd import ops
            s["workspace"] = torch.empty((ops.beam_select_workspace_size(B, W, V, n),), dtype=torch.uint8, device=DEV)
    else:
        B, W, page, width = c["B"], c["W"], c["page"], c["width"]
        pages = _pages(c)
        order = torch.randperm(pages, generator=g, device=DEV).tolist()
        refs, rows, lens = [0] * pages, [], []
        for b in range(B):
            prompt = rng.randint(max(1, c["prompt"] // 2), c["prompt"])
            shared = [order.pop() for _ in range(prompt // page)]        # full pages of the prompt
            new = rng.randint(0, c["most"])                              # tokens since, the same number in each row
            length = prompt + new
            for _ in range(W):
                row = shared + [order.pop() for _ in range((length + page - 1) // page - len(shared))]
                for p in row:
                    refs[p] += 1
                rows.append(row + [-1] * (width - len(row)))
                lens.append(length)
        s["table"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["refs"] = torch.tensor(refs, dtype=torch.int32, device=DEV)
        # a few rows go on more often than others; one in fifty ends
        picks = [[-1 if rng.random() < 0.02 else min(rng.randrange(W), rng.randrange(W)) for _ in range(W)] for _ in range(B)]
        s["parents"] = torch.tensor(picks, dtype=torch.int32, device=DEV)
        s["caches"] = [randn(pages, page, c["Hkv"], c["D"]).to(dt) for _ in range(c["tensors"])]
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from forge_amd import ops
    c = s["case"]
    if c["kind"] == "store":
        ops.cache4_write(s["k"], s["v"], s["cache"], s["slots"])
        return ops.cache4_read(s["cache"], s["slots"], c["D"], _dtype(c), k_out=s["k_out"], v_out=s["v_out"])
    if c["kind"] == "attend":
        return ops.cache4_attention(s["q"], s["cache"], s["table"], s["lens"], tree=s["tree"], workspace=s["workspace"],
                                    out=s["out"])
    if c["kind"] == "beams":
        return ops.beam_select(s["logits"], s["scores"], c["count"], ended=s["ended"], end_token=s["end"],
                               workspace=s["workspace"], out=s["out"])
    forked = ops.fork_pages(s["table"], s["lens"], s["parents"], s["refs"], c["page"])
    ops.copy_pages(s["caches"], forked.src, forked.dst)
    return (forked.table, forked.lens, forked.refs, forked.slots, forked.src, forked.dst, *s["caches"])


def _softmax_rows(scores, seen):
    """Row softmax over the seen entries; rows that see nothing are zeros."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _values(n, numbers):
    """(.., D) integers and (.., 2) step and lowest value -> what they stand for, in 32 bits."""
    return n.float() * numbers[..., :1].float() + numbers[..., 1:].float()


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "store":
        D, page, dt = c["D"], c["page"], _dtype(c)
        kb, vb, numbers = _parts(s["cache"], page, D)
        p, r = s["slots"].long() // page, s["slots"].long() % page
        for x, put in ((s["k"], 0), (s["v"], 1)):
            n, step, low = _quantize(x)
            if put == 0:
                kb[p, :, r] = _pack(n, D)
            else:
                vb[p, :, r // 4, :, r % 4] = _pack(n, D)
            numbers[p, :, r, 2 * put:2 * put + 2] = torch.stack([step, low], -1).view(torch.uint8).view(*n.shape[:2], 2, 2)
        num = numbers[p, :, r].contiguous().view(dt).view(c["T"], c["Hkv"], 4)
        return (_values(_unpack(kb[p, :, r], D), num[..., :2]).to(dt),
                _values(_unpack(vb[p, :, r // 4, :, r % 4], D), num[..., 2:]).to(dt))
    if c["kind"] == "attend":
        return _attend_plain(s)
    if c["kind"] == "beams":
        return _beams_plain(s)
    return _fork_plain(s)


def _attend_plain(s):
    c, dt = s["case"], _dtype(s["case"])
    T, Hkv, D, page = c["T"], c["Hkv"], c["D"], c["page"]
    group, scale = c["Hq"] // Hkv, 1.0 / math.sqrt(D)
    kb, vb, numbers = _parts(s["cache"], page, D)
    out = torch.empty_like(s["out"])
    j = torch.arange(T, device=DEV)
    for b, L in enumerate(_lens(c)):
        pages = s["table"][b, :(L + T + page - 1) // page].long()
        num = numbers[pages].contiguous().view(dt).view(len(pages), Hkv, page, 4)
        k = _values(_unpack(kb[pages], D), num[..., :2])                  # page, head, position, dim
        v = _values(_unpack(vb[pages].transpose(3, 4).flatten(2, 3), D), num[..., 2:])
        k = k.permute(1, 3, 0, 2).flatten(2)[..., :L + T].contiguous()    # head, dim, key
        v = v.permute(1, 0, 2, 3).flatten(1, 2)[:, :L + T].contiguous()   # head, key, dim
        q = s["q"][b].float().view(T, Hkv, group, D).permute(1, 0, 2, 3).reshape(Hkv, T * group, D)
        if s["tree"] is None:
            drafts = j[None, :] <= j[:, None]
        else:
            drafts = ((s["tree"][b][:, None] >> j) & 1) == 1
        seen = torch.cat([torch.ones((T, L), dtype=torch.bool, device=DEV), drafts], dim=1).repeat_interleave(group, 0)
        o = _softmax_rows(torch.matmul(q, k) * scale, seen) @ v
        out[b] = o.view(Hkv, T, group, D).permute(1, 0, 2, 3).reshape(T, c["Hq"], D).to(dt)
    return out


def _beams_plain(s):
    c = s["case"]
    B, W, V, count = c["B"], c["W"], c["V"], c["count"]
    x = s["logits"].double()                                       # in 64 bits: neighbours may differ in the last place only
    top = x.amax(-1, keepdim=True)
    score = x - (top + torch.exp(x - top).sum(-1, keepdim=True).log()) + s["scores"].double()[..., None]
    if s["ended"] is not None:
        score = torch.where(s["ended"][..., None], float("-inf"), score)
        score[..., s["end"]] = torch.where(s["ended"], s["scores"].double(), score[..., s["end"]])
    score, at = score.flatten(1).sort(dim=-1, descending=True, stable=True)
    score, at = score[:, :count], at[:, :count]
    none = ~(score > float("-inf"))
    short = count - score.shape[1]                                  # more places than W V
    fill = torch.nn.functional.pad
    return (fill(score.masked_fill(none, float("-inf")).float(), (0, short), value=float("-inf")),
            fill((at // V).masked_fill(none, -1).to(torch.int32), (0, short), value=-1),
            fill((at % V).masked_fill(none, -1).to(torch.int32), (0, short), value=-1))


def _fork_plain(s):
    c = s["case"]
    page, width, W, R = c["page"], c["width"], c["W"], c["B"] * c["W"]
    table, refs = s["table"].long(), s["refs"].long()
    row = torch.arange(R, device=DEV)
    local = s["parents"].flatten().long()
    on = (local >= 0) & (local < W)
    parent = torch.where(on, row // W * W + local, 0)
    lens = torch.where(on, s["lens"].long()[parent], 0)
    at = lens // page                                               # the page of the next token
    new = torch.where(on[:, None] & (torch.arange(width, device=DEV) < at[:, None]), table[parent], -1)
    room = on & (at < width)
    last = torch.where(room, table[parent, at.clamp_max(width - 1)], -1)
    first = torch.full((R,), R, device=DEV).scatter_reduce(0, parent[on], row[on], "amin")
    keep = room & (last >= 0) & (first[parent] == row) & (refs[last.clamp_min(0)] == 1)
    take = room & ~keep
    free = (refs == 0).nonzero().flatten()
    rank = take.cumsum(0) - 1
    got = take & (rank < len(free))
    fresh = torch.where(got, torch.nn.functional.pad(free, (0, 1))[rank.clamp(0, len(free))], -1)
    mine = torch.where(keep, last, fresh)
    new[row[room], at[room]] = mine[room]
    slots = torch.where(room & (mine >= 0), mine * page + lens % page, -1)
    copied = got & (lens % page > 0) & (last >= 0)
    src, dst = torch.where(copied, last, -1), torch.where(copied, fresh, -1)
    old = table[table >= 0]
    now = new[new >= 0]
    refs = refs.index_add(0, old, -torch.ones_like(old)).index_add(0, now, torch.ones_like(now))
    for t in s["caches"]:
        t[dst[copied]] = t[src[copied]]
    return tuple(x.to(torch.int32) for x in (new, lens, refs, slots, src, dst)) + tuple(s["caches"])


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; a multiply-add is two operations."""
    c = case
    if c["kind"] == "store":
        # 16-bit values in and out, 4-bit values with two numbers a head written and read
        values = 2 * c["T"] * c["Hkv"] * c["D"]
        return {"bytes": 4 * values + values + 16 * c["T"] * c["Hkv"] + 8 * c["T"], "flops": 6 * values}
    if c["kind"] == "attend":
        lens, T = _lens(c), c["T"]
        keys = sum(n + T for n in lens)
        return {"bytes": keys * c["Hkv"] * (c["D"] + 8) + 4 * len(lens) * T * c["Hq"] * c["D"]
                + (8 * len(lens) * T if T > 1 else 0) + 4 * len(lens) + 4 * sum((n + T + c["page"] - 1) // c["page"] for n in lens),
                "flops": 4 * c["D"] * c["Hq"] * T * keys}
    if c["kind"] == "beams":
        n = c["B"] * c["W"] * c["V"]
        return {"bytes": n * (4 if c["dtype"] == "float32" else 2) + 12 * c["B"] * c["count"] + 5 * c["B"] * c["W"], "flops": 3 * n}
    # tables and counts once each way, and about half of the rows' last pages
    R = c["B"] * c["W"]
    return {"bytes": 8 * R * c["width"] + 8 * _pages(c) + 24 * R + R // 2 * 4 * c["tensors"] * c["page"] * c["Hkv"] * c["D"],
            "flops": 2 * R * c["width"]}


# ---- the same results in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _store_exact, "attend": _attend_exact, "beams": _beams_exact, "fork": _fork_exact}[case["kind"]](s)


def _store_exact(s):
    dt = _dtype(s["case"])

    def held(x):
        x = x.double()
        low, top = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # the definition takes the step from two quotients of 32 bits: each is the 64-bit one rounded once
        want = ((top / torch.full_like(top, 15.0)).float() - (low / torch.full_like(low, 15.0)).float()).double()
        bits = 11 if dt == torch.float16 else 8
        unit = torch.exp2((torch.floor(torch.log2(want.clamp_min(1e-300))) + 1 - bits).clamp_min(-24.0 if bits == 11 else -133.0))
        step = torch.floor(want / unit) * unit
        n = torch.where(step > 0, torch.round((x - low) / step.clamp_min(1e-300)), 0.0).clamp(max=15.0)
        return (low + n * step).float().to(dt).double()                    # read back in 16 bits
    return held(s["k"]), held(s["v"])


def _attend_exact(s):
    c = s["case"]
    T, Hkv, D, page = c["T"], c["Hkv"], c["D"], c["page"]
    group, dt, W = c["Hq"] // Hkv, _dtype(c), _words(D)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    d = torch.arange(D, device=DEV)
    word, bit = d // 8, 4 * (d % 8 // 2) + 16 * (d % 2)
    for b, L in enumerate(_lens(c)):
        at = torch.arange(L + T, device=DEV)
        p, r = s["table"][b].long()[at // page], at % page
        if T == 1:
            hidden = torch.zeros((1, L + 1), dtype=torch.float64, device=DEV)
        else:
            bits = [[0.0 if (m >> t) & 1 else -math.inf for t in range(T)] for m in s["tree"][b].tolist()]
            hidden = torch.zeros((T, L + T), dtype=torch.float64, device=DEV)
            hidden[:, L:] = torch.tensor(bits, dtype=torch.float64, device=DEV)
        for h in range(Hkv):
            rows = s["cache"][:, h].flatten(1)[p]                           # key, bytes of its page
            at_k = (r[:, None] * W + word) * 4 + bit // 8
            at_v = page * 4 * W + ((r[:, None] // 4 * W + word) * 4 + r[:, None] % 4) * 4 + bit // 8
            num = rows.gather(1, page * 8 * W + 8 * r[:, None] + torch.arange(8, device=DEV)).view(dt).double()
            k = ((rows.gather(1, at_k) >> (bit % 8)) & 15).double() * num[:, :1] + num[:, 1:2]
            v = ((rows.gather(1, at_v) >> (bit % 8)) & 15).double() * num[:, 2:3] + num[:, 3:]
            for hq in range(h * group, (h + 1) * group):
                z = s["q"][b, :, hq].double() @ k.T.contiguous() / math.sqrt(D) + hidden
                out[b, :, hq] = torch.softmax(z, -1) @ v
    return out


def _beams_exact(s):
    """One place after the other: the largest score that is left, the first of equal ones."""
    c = s["case"]
    B, V = c["B"], c["V"]
    flat = (torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None])
    if s["ended"] is not None:
        flat[s["ended"]] = float("-inf")
        for b, w in s["ended"].nonzero().tolist():
            flat[b, w, s["end"]] = s["scores"][b, w].double()
    flat = flat.flatten(1)
    places = torch.arange(flat.shape[1], device=DEV)
    scores, beams, tokens = [], [], []
    for _ in range(c["count"]):
        best = flat.amax(-1)
        at = torch.where(flat == best[:, None], places, flat.shape[1]).amin(-1)
        some = best > float("-inf")
        scores.append(best)
        beams.append(torch.where(some, at // V, -1))
        tokens.append(torch.where(some, at % V, -1))
        flat[torch.arange(B, device=DEV), at] = float("-inf")
    return torch.stack(scores, -1), torch.stack(beams, -1).to(torch.int32), torch.stack(tokens, -1).to(torch.int32)


def _fork_exact(s):
    """Row by row on the host."""
    c = s["case"]
    page, width, W = c["page"], c["width"], c["W"]
    table, lens, refs, parents = (s[k].tolist() for k in ("table", "lens", "refs", "parents"))
    counts = list(refs)
    for row in table:
        for p in row:
            if p >= 0:
                counts[p] -= 1
    free = [p for p, n in enumerate(refs) if n == 0]
    new, new_lens, slots, src, dst, seen = [], [], [], [], [], set()
    for r in range(len(table)):
        up = parents[r // W][r % W]
        fresh_row, slot, a, b, length = [-1] * width, -1, -1, -1, 0
        if 0 <= up < W:
            up += r // W * W
            length = lens[up]
            at, first = length // page, up not in seen
            seen.add(up)
            fresh_row[:at] = table[up][:at]
            if at < width:
                mine = last = table[up][at]
                if not (first and last >= 0 and refs[last] == 1):
                    mine = free.pop(0) if free else -1
                    if mine >= 0 and length % page and last >= 0:
                        a, b = last, mine
                fresh_row[at] = mine
                if mine >= 0:
                    slot = mine * page + length % page
        new.append(fresh_row)
        new_lens.append(length)
        slots.append(slot)
        src.append(a)
        dst.append(b)
        for p in fresh_row:
            if p >= 0:
                counts[p] += 1
    caches = []
    for t in s["caches"]:
        t = t.clone()
        pairs = [(a, b) for a, b in zip(src, dst) if b >= 0]
        if pairs:
            a, b = (torch.tensor(x, device=DEV) for x in zip(*pairs))
            t.index_copy_(0, b, t.index_select(0, a))
        caches.append(t)
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (new, new_lens, counts, slots, src, dst)) + tuple(caches)
