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
