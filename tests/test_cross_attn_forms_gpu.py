"""The form that kiln_cross_attn runs is the one that its sizes and its workspace say."""
import pytest
import torch

import kiln_amd as ka
from tests.test_cross_attn_gpu import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", [(20, 1, 77, 16, 16, 128), (20, 1, 100, 16, 16, 64), (17, 2, 128, 32, 16, 128), (25, 1, 32, 16, 16, 64),
                                               (4, 1, 512, 16, 16, 128), (2, 300, 200, 8, 8, 64)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_no_workspace_needed(gpu, B, Tq, Tk, Hq, Hkv, Dh, dt):
    """Sizes that need no workspace: with none, an empty one and one that is not needed, the same form, and the same bits. The first
    four have more key heads than CUs, less than two for each: a wave alone for all keys of one."""
    assert ka.cross_attn_workspace_bytes(B, Tq, Tk, Hq, Hkv, Dh) == 0
    if B > 4:
        assert ka.cross_attn_form(B, Tq, Tk, Hq, Hkv, Dh) == (16, 1, False)
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, dt)
    outs = [ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv, workspace=ws)
            for ws in (None, torch.empty(0, dtype=torch.uint8, device=DEV), torch.empty(1 << 20, dtype=torch.uint8, device=DEV))]
    check(outs[0], q, k, v, Hq, Hkv, what=f"{B} {Tq} {Tk} {Hq} {Hkv} {Dh} {dt}")
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
