"""The largest 4-bit caches: 2^31 positions are taken, and one page more is refused."""
import ctypes

import pytest

from helpers import say

FAKE = ctypes.c_void_p(4096)    # never dereferenced: there is no device


def test_positions():
    """Without a device, a call that passes the checks comes back with the runtime's error and not with that of its arguments."""
    import torch
    if torch.cuda.device_count():
        pytest.skip("made-up addresses: only where nothing can be launched")
    import forge_amd
    lib = forge_amd.load()
    for page in (16, 4096, 1 << 20):
        for pages, ok in (((1 << 31) // page, True), ((1 << 31) // page + 1, False)):
            codes = [lib.forge_cache4_write(FAKE, FAKE, FAKE, FAKE, 3, 2, 64, pages, page, 128, 64, 128, 64, 0, None),
                     lib.forge_cache4_read(FAKE, FAKE, FAKE, FAKE, 3, 2, 64, pages, page, 0, None),
                     lib.forge_cache4_attention(FAKE, FAKE, FAKE, FAKE, None, FAKE, 1, 1, 2, 2, 64, pages, page, 1, 0.1, 0, FAKE, 1 << 40, None)]
            assert all((code > 0) if ok else code == -1 for code in codes), (page, pages, codes)


@pytest.mark.gpu
def test_last_positions(dev):
    """The last page of a cache of 2^31 positions is written, read and attended to as that of a cache of one page."""
    import torch
    from forge_amd import ops
    from test_gpu_cache4 import heads, stored
    page, D = 4096, 64
    pages = (1 << 31) // page
    shape = ops.cache4_shape(pages, page, 1, D)
    if torch.cuda.mem_get_info()[0] < pages * shape[2] * shape[3] + (1 << 33):
        pytest.skip("a cache of 155 GB")
    say("cache4 of 2^31 positions")
    cache = torch.empty(shape, dtype=torch.uint8, device=dev)
    small = torch.empty(ops.cache4_shape(1, page, 1, D), dtype=torch.uint8, device=dev)
    k, v, q = heads(page, 1, D, "float16", dev, 1), heads(page, 1, D, "float16", dev, 2), heads(1, 4, D, "float16", dev, 3)[None]
    at = torch.arange(page, dtype=torch.int32, device=dev)
    slots = at + ((1 << 31) - page)
    ops.cache4_write(k, v, cache, slots)
    ops.cache4_write(k, v, small, at)
    rk, rv = ops.cache4_read(cache, slots, D)
    assert torch.equal(rk, stored(k, D, "float16")) and torch.equal(rv, stored(v, D, "float16"))
    lens = torch.tensor([page - 1], dtype=torch.int32, device=dev)
    out = [ops.cache4_attention(q, c, torch.tensor([[n]], dtype=torch.int32, device=dev), lens) for c, n in ((cache, pages - 1), (small, 0))]
    assert torch.isfinite(out[0]).all() and torch.equal(*out)
    del cache
    torch.cuda.empty_cache()


def test_requests_of_a_grid():
    """A grid's dimension has under 2^32 threads: of 512 to a request and of 256 to a piece. More is refused."""
    import forge_amd
    size = forge_amd.load().forge_beam_select_workspace_size
    assert size((1 << 23) - 1, 1, 10, 1) > 0 and size(1 << 23, 1, 10, 1) == 0
    assert size((1 << 14) - 1, 1024, 8192, 1) > 0 and size(1 << 14, 1024, 10, 1) == 0
    assert size(1 << 13, 1000, 16384, 4) > 0 and size(1 << 13, 1000, 16385, 4) == 0


@pytest.mark.gpu
def test_more_requests_than_a_grid(dev):
    import torch
    from forge_amd import ops
    x = torch.zeros((1, 1, 8), dtype=torch.float16, device=dev).expand((1 << 23) + 5, 1, 8)
    with pytest.raises(ValueError, match="more than one call"):
        ops.beam_select(x, torch.zeros((x.shape[0], 1), device=dev), 1)


@pytest.mark.gpu
def test_more_tokens_than_a_grid(dev):
    """2^24 workgroups and a few: each token's slot takes it, and reads it back."""
    import torch
    from forge_amd import ops
    from test_gpu_cache4 import heads, stored
    H, D, T, page = 64, 8, (1 << 23) + 1000, 16
    say(f"cache4_write of {T} tokens of {H} heads")
    base = heads(1, H, D, "float16", dev, 5)
    cache = torch.zeros(ops.cache4_shape(2, page, H, D), dtype=torch.uint8, device=dev)
    slots = torch.full((T,), -1, dtype=torch.int32, device=dev)
    at = torch.tensor([0, 1, 77, (1 << 22) + 5, T - 1200, T - 1009, T - 33, T - 2, T - 1], device=dev)
    slots[at] = torch.arange(at.numel(), dtype=torch.int32, device=dev) * 3
    ops.cache4_write(base.expand(T, H, D), -base.expand(T, H, D), cache, slots)
    k, v = ops.cache4_read(cache, torch.arange(32, dtype=torch.int32, device=dev), D)
    live = torch.zeros(32, dtype=torch.bool, device=dev)
    live[slots[at].long()] = True
    for got, want in ((k, stored(base, D, "float16")), (v, stored(-base, D, "float16"))):
        assert torch.equal(got[live], want.expand(at.numel(), H, D)) and (got[~live] == 0).all()
    k, v = ops.cache4_read(cache, slots, D)
    for got, want in ((k, stored(base, D, "float16")), (v, stored(-base, D, "float16"))):
        assert torch.equal(got[at], want.expand(at.numel(), H, D)) and int((got != 0).any(-1).any(-1).sum()) == at.numel()
    del k, v, got
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_largest_page(dev):
    """A page of more than 2^24 pieces of 4 KB."""
    import torch
    from forge_amd import ops
    n = (1 << 36) + 4096 * 3 + 16
    if torch.cuda.mem_get_info()[0] < 2 * n + (1 << 33):
        pytest.skip("pages of 69 GB")
    say(f"copy_pages of {n} bytes")
    cache = torch.empty((2, n), dtype=torch.uint8, device=dev)
    cache[1].zero_()
    at = [0, 4095, 4096, (1 << 32) - 1, 1 << 32, (1 << 32) + 70000, (1 << 35) + 1, (1 << 36) - 1, 1 << 36, n - 17, n - 1]
    for i, a in enumerate(at):
        cache[0, a] = i + 1
        cache[1, a] = 200
    ops.copy_pages([cache], torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev))
    assert [int(cache[1, a]) for a in at] == list(range(1, len(at) + 1))
    del cache
    torch.cuda.empty_cache()
