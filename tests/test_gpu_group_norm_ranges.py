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


@pytest.mark.parametrize('shape', [(40000, 2, 3, 8, 2), (5000, 4, 4, 64, 8), (3000, 3, 3, 35, 5)], ids=B.name)
def test_parameter_gradients_of_large_batches(cuda, shape, form):
    """The samples' partial sums (bounds of one sample) are added up without further loss: one rounding of the result."""
    from stmi import ops
    *dims, groups = shape
    gen = torch.Generator().manual_seed(5)
    n, h, w, c = dims
    x, scale, shift = torch.randn(dims, generator=gen).to(cuda), torch.ones(c, device=cuda), torch.zeros(c, device=cuda)
    # equal terms: in a running sum of 32 bits their roundings do not cancel
    dy = torch.full(dims, 0.7, device=cuda)
    _, stats = ops.group_norm_fwd(x, groups, scale, shift, eps=B.EPS)
    dscale, dshift = torch.zeros((2, c), device=cuda)
    ops.group_norm_bwd(x, dy, groups, stats, scale, shift, dscale, dshift, accumulate=False)
    want = dy.double().sum((0, 1, 2))
    # a sample's h w terms: at most h w roundings of at most u of the partial sum
    assert ((dshift.double() - want).abs() <= (h * w + 1) * U * want.abs()).all()
    mean, rstd = (stats[..., k].double().repeat_interleave(c // groups, 1).view(n, 1, 1, c) for k in (0, 1))
    terms = dy.double() * (x.double() - mean) * rstd
    assert ((dscale.double() - terms.sum((0, 1, 2))).abs() <= ((h * w + 6) * U * terms.abs().sum((0, 1, 2)))).all()


def test_parameter_gradients_of_the_samples_behind_the_first_launch(cuda):
    """131075 samples of 512 groups take several launches of one block per group.  Only the samples at their borders have
    gradients: a row that is lost or counted twice shows in full."""
    from stmi import ops
    n, c, groups = 131075, 4096, 512
    x7, scale, shift, dy7 = (t.to(cuda) for t in B.data((7, 1, 1, c), groups, torch.bfloat16, 41))
    x = x7.repeat(18725, 1, 1, 1)
    dy = torch.zeros_like(x)
    at = [0, 1, 65535, 65536, 131070, 131071, 131072, 131073, 131074]
    for k, i in enumerate(at):
        dy[i] = dy7[k % 7]
    _, stats = ops.group_norm_fwd(x, groups, scale, shift, eps=B.EPS)
    dscale, dshift = torch.zeros((2, c), device=cuda)
    dx = ops.group_norm_bwd(x, dy, groups, stats, scale, shift, dscale, dshift, accumulate=False)
    few_x, few_dy = x[at].contiguous(), dy[at].contiguous()
    want, parts = B.results(few_x, groups, scale, shift, ops.ACT_NONE, few_dy)
    assert not B.faults({'dx': dx[at], 'dscale': dscale, 'dshift': dshift}, want, B.bounds(parts), parts, torch.bfloat16)
    dx[at] = 0
    assert not dx.any()
