"""kiln_prompt_attn: values of hidden keys that are not finite, in every form, and with so many query heads on a key head that all rows of a wave
are one token's while the workgroup's other waves hold later ones."""

import math

import pytest
import torch

import kiln_amd as ka
from test_prompt_attn_gpu import DEV, NAN, Case, form_of

pytestmark = pytest.mark.gpu

# sequences (queries, keys), query heads, key heads, head size, prefix, (rows of a workgroup, how keys are shared out)
MANY_HEADS = [
    ([(200, 200), (30, 30)], 32, 1, 64, 0, (64, 0)), ([(90, 90), (7, 7)], 40, 1, 128, 33, (64, 0)), ([(200, 200), (30, 30)], 48, 1, 128, 0, (64, 0)),
    ([(90, 90), (5, 50)], 63, 1, 64, 0, (64, 0)), ([(70, 70), (7, 7)], 96, 1, 64, 33, (64, 0)), ([(9, 9)] * 3, 128, 2, 128, 0, (64, 0)),
    ([(700, 700)] * 6, 32, 1, 128, 0, (128, 0)), ([(300, 300)] * 3, 64, 1, 64, 40, (128, 0)), ([(500, 500)] * 3, 71, 1, 64, 0, (128, 0)),
    ([(500, 500)] * 4, 48, 1, 128, 0, (128, 0)),
    ([(40, 6000), (7, 100)], 64, 2, 128, 0, (64, 1)), ([(40, 6000)], 32, 1, 64, 70, (64, 1)), ([(8, 3000)] * 2, 71, 1, 64, 0, (64, 1)),
    ([(2, 30), (0, 5)] * 30, 32, 1, 64, 3000, (64, 2)), ([(2, 30), (0, 5)] * 30, 32, 1, 128, 3000, (64, 2)), ([(4, 40), (0, 5), (0, 0), (0, 1)] * 8, 32, 1, 64, 9000, (64, 2))]
FEW_HEADS = [
    ([(150, 150)] * 3, 8, 4, 128, 0, (64, 0)), ([(600, 600)] * 20, 16, 8, 64, 0, (128, 0)), ([(700, 700)] * 24, 8, 4, 128, 0, (128, 0)),
    ([(100, 4000)], 7, 1, 64, 0, (64, 1)), ([(100, 4000), (20, 60)], 4, 1, 128, 33, (64, 1)),
    ([(4, 3000), (3, 5000)], 2, 1, 64, 0, (16, 1)), ([(4, 3000), (3, 5000)], 4, 2, 128, 40, (16, 1)), ([(2, 2)] * 70, 4, 1, 64, 5000, (16, 2)),
    ([(3, 90)] * 30, 8, 4, 128, 2500, (16, 2)), ([(3, 20)] * 150, 16, 2, 128, 6000, (64, 2)), ([(3, 20)] * 150, 32, 4, 64, 6000, (64, 2))]


@pytest.mark.parametrize("bad", [math.inf, NAN])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,Dh,P,form", MANY_HEADS + FEW_HEADS)
def test_hidden_values(gpu, lens, Hq, Hkv, Dh, P, form, dt, bad):
    """Rows that do not see a value keep their bits, those that see it are not finite."""
    c = Case(lens, Hq, Hkv, Dh, dt, P=P, seed=Hq)
    assert ka.prompt_attn_form(len(lens), c.q.shape[0], c.k.shape[0], P, Hq, Hkv, Dh) == form
    c.run()
    if not math.isnan(bad):  # (clean inputs: once)
        c.check(f"clean {Hq}/{Hkv} of {Dh} P={P}")
    clean, k, v = c.out.clone(), c.k.clone(), c.v.clone()
    G, n = Hq // Hkv, c.q.shape[0]
    # single values of V: of the second query's own key, one in the middle, the last; and then whole tokens of K and V
    values, tokens = torch.zeros(n, Hkv, Dh, dtype=torch.bool, device=DEV), torch.zeros(n, dtype=torch.bool, device=DEV)
    places = []
    for s, (q0, nq, k0, nk) in enumerate(c.seqs):
        for j, i in enumerate({i for i in (1, nq // 2, nq - 1) if 0 < i < nq}):
            places.append((k0 + nk - nq + i, (s + 5 * j) % Hkv, (37 * s + 11 * j) % Dh))
            values[q0 + i:q0 + nq, places[-1][1], places[-1][2]] = True
        if nq > 1:
            tokens[q0 + nq // 2:q0 + nq] = True
    for t, h, d in places:
        c.v[t, h * Dh + d] = bad
    c.out.fill_(7.0)
    c.run()
    want = values[:, :, None].expand(n, Hkv, G, Dh).reshape(n, Hq * Dh)
    assert want.any() and torch.equal(c.out[~want], clean[~want])
    assert not torch.isfinite(c.out[want]).any()
    c.k, c.v = k, v
    for q0, nq, k0, nk in c.seqs:
        if nq > 1:
            c.k[k0 + nk - nq + nq // 2], c.v[k0 + nk - nq + nq // 2] = bad, bad
    c.out.fill_(7.0)
    c.run()
    assert torch.equal(c.out[~tokens], clean[~tokens])
    assert not torch.isfinite(c.out[tokens]).any()


def test_every_form_is_reached(gpu):
    forms = {(c[3], c[5]) for c in MANY_HEADS + FEW_HEADS}
    assert forms == {(d, f) for d in (64, 128) for f in ((64, 0), (128, 0), (16, 1), (64, 1), (16, 2), (64, 2))}
