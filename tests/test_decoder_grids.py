"""CPU: decoder calls of more work than a grid has threads for (2^32 in a dimension) are refused; a launch would do a part of it and say nothing."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    import forge_amd
    return forge_amd.load()


def test_qk_norm_rope(lib):
    for T in (1 << 24, (1 << 31) - 1):
        assert lib.forge_qk_norm_rope(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, 64, T, 4, 2, 64, 64, 10,
                                      256, 64, 128, 64, 128, 64, 1e-6, 0, 0, None) == -1


@pytest.mark.parametrize("tokens,Hq,Hkv,D", [(1 << 30, 4, 4, 64), (1 << 29, 4, 4, 256), (1 << 25, 64, 64, 128)])
def test_prompt_attention(lib, tokens, Hq, Hkv, D):
    assert lib.forge_prompt_attention(FAKE, FAKE, FAKE, FAKE, FAKE, 1, tokens, Hq, Hkv, D, Hq * D, D, Hkv * D, D, Hkv * D, D, 0.1, 1, 0,
                                      None) == -1


def test_int4(lib):
    for M, K, N in ((1 << 17, 128, 1 << 15), (1, 4096, (1 << 28) + 16), (64, 512, 1 << 30)):
        assert lib.forge_int4_linear(FAKE, FAKE, FAKE, None, FAKE, M, K, N, 128, 0, None) == -1, (M, K, N)
    assert lib.forge_quantize_weight_int4(FAKE, 1, FAKE, FAKE, 1 << 26, 512, 128, None) == -1
    assert lib.forge_pack_weight_int4(FAKE, FAKE, 1 << 26, 512, None) == -1
