"""Calls of the attention section over an encoder's states that are refused before anything reaches the GPU."""
import pytest

import kiln_amd as ka

EINVAL, EUNSUP, ENOMEM = ka.KILN_EINVAL, ka.KILN_EUNSUPPORTED, ka.KILN_ENOMEM
F32, F16, BF16 = ka.KILN_F32, ka.KILN_F16, ka.KILN_BF16
P, Q, R, S = (1 << 20) * 16, (1 << 21) * 16, (1 << 22) * 16, (1 << 23) * 16  # addresses that no call below touches


@pytest.fixture(scope="module")
def L():
    return ka.lib()


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_cross_attn_scale(L, scale):
    """A scale that is finite but not in the units of log2 that the kernel works in: 0 times it would be a NaN."""
    assert L.kiln_cross_attn(P, 256, 1024, Q, 256, 1024, R, 256, 2048, S, 256, 2048, F16, 2, 4, 8, 2, 2, 128, scale, None, None, 8, None, 0,
                             None) == EINVAL
