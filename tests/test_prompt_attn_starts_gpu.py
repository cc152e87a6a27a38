"""kiln_prompt_attn: starts and lengths far outside the tensors, 32-bit integers' ends among them, are clamped, and what they clamp to is what is
computed."""

import pytest
import torch

import kiln_amd as ka
from test_prompt_attn_gpu import DEV, Case

pytestmark = pytest.mark.gpu
LO, HI = -(1 << 31), (1 << 31) - 1


@pytest.mark.parametrize("heads,P", [((4, 2, 64), 0), ((4, 2, 64), 70), ((32, 1, 128), 33), ((7, 1, 64), 0)])
@pytest.mark.parametrize("starts,ks,kl", [
    ([LO, 20, 50, HI], [LO, HI, 5], [HI, 4, LO]), ([LO, LO, HI, HI], [0, 0, 0], [HI, HI, HI]), ([0, 20, 50, 60], [HI, HI - 1, 40], [HI, 1, HI]),
    ([-1, 20, 50, 1 << 30], [3, -1, 60], [HI - 3, HI - 40, 1 << 30]), ([HI, HI, HI, HI], [0, 0, 0], [5, 5, 5]), ([LO, -5, 0, 64], [LO, LO, LO], [LO, -1, HI])])
@pytest.mark.parametrize("split", [False, True])
def test_clamped(gpu, starts, ks, kl, heads, P, split):
    lens = [(20, 20), (30, 30), (10, 9000 if split else 10)]
    c = Case(lens, *heads, torch.float16, pad=4, cached=True, P=P)
    form = ka.prompt_attn_form(3, c.q.shape[0], c.k.shape[0], P, *heads)
    assert form[1] == int(split), form
    n, m = c.q.shape[0], c.k.shape[0]
    for t, values in ((c.q_start, starts), (c.k_start, ks), (c.k_len, kl)):
        t.copy_(torch.tensor(values, dtype=torch.int32))
    c.k.nan_to_num_(0.5)
    c.v.nan_to_num_(0.5)
    at = [min(max(s, 0), n) for s in starts]
    c.seqs = []
    for a, b, s, l in zip(at, at[1:], ks, kl):
        s = min(max(s, 0), m)
        c.seqs.append((a, b - a, s, min(max(l, 0), m - s)))
    c.run()
    c.check(f"{starts} {ks} {kl}")
