"""INT8 calls of more work than a grid has threads for (2^32 in a dimension): done in several launches, or refused; a launch would do a part of it
and say nothing."""
import ctypes

import pytest

from helpers import say

FAKE = ctypes.c_void_p(4096)    # never dereferenced: validation fails first
BYTE = ctypes.c_void_p(4097)


def test_refused():
    import forge_amd
    lib = forge_amd.load()
    big = 1 << 24
    assert lib.forge_quantize_activation_twopass(FAKE, FAKE, FAKE, big, 64, 256, None) == -1
    assert lib.forge_quantize_activation_twopass(FAKE, FAKE, FAKE, big // 4, 64, 1024, None) == -1
    assert lib.forge_dequantize_bias(FAKE, FAKE, FAKE, None, FAKE, big, 5, None) == -1
    assert lib.forge_quantize_weight_rows(FAKE, 1, FAKE, FAKE, big, 64, None) == -1
    assert lib.forge_prepare_sparse_weight(FAKE, 1, FAKE, FAKE, FAKE, big, 64, None) == -1
    assert lib.forge_prune_compress_24(BYTE, FAKE, FAKE, 1 << 30, 16, None) == -1
    assert lib.forge_pack_metadata(BYTE, FAKE, 1 << 30, 128, None) == -1
    # 2^26 planes of a wave each, four waves to a workgroup
    assert lib.forge_int8_depthwise_conv2d_forward(FAKE, FAKE, FAKE, None, FAKE, 1 << 16, 1 << 10, 8, 8, 3, 3, 1, 1, 1, 1, 1, 1, None) == -1


@pytest.mark.gpu
def test_quantized_rows(dev):
    """Four rows to a workgroup and 2^26 of them, and a few: every row, those around the launches' ends against the same rows alone."""
    import torch
    from forge_amd import ops
    M, K = (1 << 26) + 777, 8
    say(f"quantize {M} x {K}")
    x = torch.randn((1 << 20, K), generator=torch.Generator().manual_seed(1)).half().to(dev).repeat((M >> 20) + 1, 1)[:M].contiguous()
    for size, dt in ((M * K, torch.int8), (M, torch.float32)):      # (what an output would hold that nobody writes)
        torch.zeros(size, dtype=dt, device=dev)
    q, s = ops.fused_quantize_activation(x, M, K)
    q, s = q.view(M, K), s.view(M)
    assert (s > 0).all()
    for at in (0, (1 << 23) - 3, (1 << 24) - 5, (1 << 26) - 3000, M - 2500):
        qa, sa = ops.fused_quantize_activation(x[at:at + 2500].contiguous(), 2500, K)
        assert torch.equal(q[at:at + 2500], qa.view(2500, K)) and torch.equal(s[at:at + 2500], sa.view(2500))
