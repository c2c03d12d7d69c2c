"""CPU: the largest sizes of cache_attention: what its kernels divide and address stays in range, or the call is refused
before a device is touched."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    import forge_amd
    return forge_amd.load()


def call(lib, B=1, T=1, Hq=8, Hkv=1, D=64, page=16, width=64):
    return lib.forge_cache_attention(FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, B, T, Hq, Hkv, D, 100, page, width, 0.1, 0, FAKE,
                                     1 << 62, None)


@pytest.mark.parametrize("sizes", [dict(Hq=1 << 16), dict(Hq=1 << 17), dict(T=64, Hq=1 << 13), dict(Hq=1 << 20, Hkv=4),
                                   dict(Hq=1 << 24, Hkv=1 << 14), dict(B=1 << 20, Hq=1 << 11), dict(width=(1 << 23) + 1)])
def test_out_of_range(lib, sizes):
    assert call(lib, **sizes) == -1
    s = dict(dict(B=1, T=1, Hq=8, Hkv=1, D=64, page=16, width=64), **sizes)
    assert lib.forge_cache_attention_workspace_size(s["B"], s["T"], s["Hq"], s["Hkv"], s["D"], s["page"] * s["width"]) == 0


@pytest.mark.parametrize("keys", [(1 << 27) - 2048, (1 << 27) - 128, (1 << 27) - 1, 1 << 27])
def test_longest_tables(lib, keys):
    """Up to 2^27 positions, in no more chunks than a grid has rows, of no more keys than a chunk's page table has place for."""
    row = (64 + 2) * 4
    size = lib.forge_cache_attention_workspace_size(1, 1, 1, 1, 64, keys)
    assert size % row == 0 and 1 < size // row <= 65535
    assert -(-keys // (size // row)) <= 2048 + 128
    assert lib.forge_cache_attention_workspace_size(1, 1, 1, 1, 64, (1 << 27) + 1) == 0
