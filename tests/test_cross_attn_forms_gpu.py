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


@pytest.mark.parametrize("Tq,Hq,Hkv,Dh,Tk", [(1, 2, 2, 64, 3000), (1, 4, 1, 128, 3000), (3, 16, 4, 128, 1000), (40, 2, 2, 64, 3000), (40, 2, 2, 128, 3000),
                                             (600, 16, 16, 128, 1100), (1500, 16, 16, 64, 1100)])
@pytest.mark.parametrize("small", [False, True])
def test_one_key_of_a_long_mask(gpu, Tq, Hq, Hkv, Dh, Tk, small):
    """An item's mask keeps one key, next to the ends of the mask's windows of 512 keys among others: its value, exactly. Keys that
    another window's bits would keep hold other values."""
    at = [i for i in (0, 1, 31, 32, 63, 64, 511, 512, 513, 767, 1000, 1023, 1024, 1055, 1535, 1536, 2047, 2048, 2560, Tk - 1) if i < Tk]
    B = len(at)
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, torch.float16)
    kmask = torch.zeros(B, Tk, dtype=torch.bool, device=DEV)
    kmask[range(B), at] = True
    want = v[range(B), at].view(B, 1, Hkv, 1, Dh).expand(B, Tq, Hkv, Hq // Hkv, Dh).reshape(B, Tq, Hq * Dh)
    ws = torch.empty(16, dtype=torch.uint8, device=DEV) if small else None
    out = ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv, kmask=kmask, workspace=ws)
    assert torch.equal(out, want)
