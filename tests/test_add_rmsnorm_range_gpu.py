"""kiln_add_rmsnorm at the borders of fp32's range: sums of squares next to the largest value, small values beside ones whose squares overflow,
and the smallest eps."""

import pytest
import torch

import kiln_amd as ka
from test_add_rmsnorm_gpu import DEV, norm_rel, reference

pytestmark = pytest.mark.gpu
DIMS = [64, 500, 1024, 2048, 4096, 20000]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("off", [0.0, 2.0 ** -23, -2.0 ** -23])
def test_sums_of_squares_next_to_the_largest(gpu, dim, off):
    """Rows of unequal values whose squares sum to fp32's largest value, give or take its last places."""
    g = torch.Generator(device=DEV).manual_seed(dim)
    x = torch.randn(500, dim, generator=g, device=DEV, dtype=torch.float64)
    x = (x * ((1 + off) * torch.finfo(torch.float32).max / (x * x).sum(-1, keepdim=True)).sqrt()).float()
    y = torch.empty_like(x)
    ka.add_rmsnorm(y, x)
    ref = reference(x, None, None)[1]
    assert ((y.double() - ref).abs() <= norm_rel(dim) * ref.abs() + 2.0 ** -149).all()


@pytest.mark.parametrize("dim", DIMS)
def test_small_values_beside_the_largest(gpu, dim):
    """Values down to where their result leaves fp32's normal range keep their relative accuracy."""
    g = torch.Generator(device=DEV).manual_seed(dim)
    x = torch.randn(40, dim, generator=g, device=DEV) * torch.exp2(torch.randint(-64, 1, (40, dim), generator=g, device=DEV).float())
    x[:, 3] = 2.0 ** torch.linspace(64, 127, 40, device=DEV)
    y = torch.empty_like(x)
    ka.add_rmsnorm(y, x)
    ref = reference(x, None, None)[1]
    assert ((y.double() - ref).abs() <= norm_rel(dim) * ref.abs() + 2.0 ** -149).all()


@pytest.mark.parametrize("dim", DIMS)
def test_small_eps(gpu, dim):
    """Squares below fp32's normal range count where eps does not exceed them; with an eps of 0.5 to 2 times their mean; rows of zeros."""
    g = torch.Generator(device=DEV).manual_seed(dim)
    for e in (-149, -148, -140, -130, -126, -110, -101, -99):
        eps = 2.0 ** e
        x = torch.randn(4, dim, generator=g, device=DEV, dtype=torch.float64) * 2.0 ** (e / 2)
        x = (x * torch.tensor([[0.7], [1.4], [0.0], [2.0 ** 60]], dtype=torch.float64, device=DEV)).float()
        y = torch.empty_like(x)
        ka.add_rmsnorm(y, x, eps=eps)
        ref = reference(x, None, None, eps)[1]
        assert ((y.double() - ref).abs() <= norm_rel(dim) * ref.abs() + 2.0 ** -149).all(), e


@pytest.mark.parametrize("dim", DIMS)
def test_large_eps(gpu, dim):
    """An eps next to the mean of squares that overflow in the sum."""
    g = torch.Generator(device=DEV).manual_seed(dim)
    x = (torch.randn(6, dim, generator=g, device=DEV, dtype=torch.float64) * (2.0 ** torch.linspace(126, 140, 6, device=DEV)[:, None].double()).sqrt()).float()
    y = torch.empty_like(x)
    for eps in (1e30, 1e37, 1e38, 3e38):
        ka.add_rmsnorm(y, x, eps=eps)
        ref = reference(x, None, None, eps)[1]
        assert ((y.double() - ref).abs() <= norm_rel(dim) * ref.abs() + 2.0 ** -149).all(), eps
