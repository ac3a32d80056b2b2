"""Group norm of very large values and of very large batches."""
import pytest
import torch

import group_norm_bounds as B

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(params=['chosen', 'slices'])
def form(request, monkeypatch):
    if request.param == 'slices':
        monkeypatch.setenv('STMI_NO_GN_UNITS', '1')


RANGE_SHAPES = [(2, 32, 32, 16, 4), (2, 16, 16, 512, 32), (1, 90, 100, 32, 2), (2, 13, 27, 35, 5), (2, 12, 9, 513, 1), (1, 3, 1, 35, 7), (1, 200, 200, 128, 128)]


@pytest.mark.parametrize('value', [1e36, -3e38, 1e30, 7.0])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('shape', RANGE_SHAPES, ids=B.name)
def test_groups_of_one_value_of_any_size(cuda, shape, dtype, value, form):
    """Equal values have no deviation: y is the shift exactly, and rstd 1 / sqrt(eps)."""
    from stmi import ops
    *dims, groups = shape
    x = torch.full(dims, value, dtype=dtype, device=cuda)
    scale, shift = torch.linspace(0.5, 1.5, dims[3], device=cuda), torch.linspace(-1, 1, dims[3], device=cuda)
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, eps=B.EPS)
    assert torch.equal(y, shift.to(dtype).expand(dims))
    assert (stats[..., 0] == x.flatten()[0].float()).all()
    assert (stats[..., 1] * B.EPS ** 0.5 - 1).abs().max() <= 4 * U
    dx = ops.group_norm_bwd(x, torch.ones_like(x), groups, stats, scale, shift, None, None)
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize('mean', [0.0, 1e20])
@pytest.mark.parametrize('shape', RANGE_SHAPES, ids=B.name)
def test_deviations_up_to_the_stated_size(cuda, shape, mean, form):
    """Deviations of up to 1e18 from the group's mean: the bounds are relative ones and hold as they stand."""
    from stmi import ops
    *dims, groups = shape
    gen = torch.Generator().manual_seed(3)
    x = mean + (torch.rand(dims, generator=gen) * 2 - 1) * 0.5e18
    scale, shift, dy = 1 + 0.2 * torch.randn(dims[3], generator=gen), 0.2 * torch.randn(dims[3], generator=gen), torch.randn(dims, generator=gen) + 1
    v = x.double().view(dims[0], -1, groups, dims[3] // groups)
    assert (v - v.mean((1, 3), keepdim=True)).abs().max() <= 1e18
    x, scale, shift, dy = (t.to(cuda) for t in (x, scale, shift, dy))
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, act=ops.ACT_SILU, eps=B.EPS)
    dscale, dshift = torch.zeros((2, dims[3]), device=cuda)
    dx = ops.group_norm_bwd(x, dy, groups, stats, scale, shift, dscale, dshift, act=ops.ACT_SILU)
    want, parts = B.results(x, groups, scale, shift, ops.ACT_SILU, dy)
    bound = B.bounds(parts)
    # dx is of the size of 1e-18: its terms are formed from numbers above 2^-126, k2 = rstd^2 m2 (1e-36) to 2^-149
    bound['dx'] = bound['dx'] + 2.0 ** -148 * 1e18
    assert not B.faults({'y': y, 'dx': dx, 'dshift': dshift, 'dscale': dscale}, want, bound, parts, torch.float32)
