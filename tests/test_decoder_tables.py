"""CPU: DecoderAttention's position tables."""
import math

import torch


def test_tables_hold_far_positions():
    """Cosines and sines of every position are those of the exact angle, rounded once to FP32."""
    from forge_amd.nn import DecoderAttention
    positions, D, theta = 131072, 32, 500000.0
    block = DecoderAttention(128, 4, 2, D, positions, theta=theta)
    assert block.cos.shape == block.sin.shape == (positions, D // 2) and block.cos.dtype == torch.float32
    for p in (0, 1, 4095, 65537, positions - 1):
        for i in range(D // 2):
            angle = p * theta ** (-2.0 * i / D)
            # half a unit of FP32 at one, and the 64-bit angle's own error
            bound = 2.0 ** -25 + angle * 2.0 ** -50
            assert abs(block.cos[p, i].item() - math.cos(angle)) <= bound
            assert abs(block.sin[p, i].item() - math.sin(angle)) <= bound
