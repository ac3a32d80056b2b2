"""Group norm, every form of the kernels, within bounds that a missing term, slice or pixel breaks (group_norm_bounds.py)."""
import pytest
import torch

import group_norm_bounds as B

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


@pytest.fixture(params=['chosen', 'slices'])
def form(request, monkeypatch):
    """The form the library chooses (small samples: one block per group), and the one that cuts samples into slices."""
    if request.param == 'slices':
        monkeypatch.setenv('STMI_NO_GN_UNITS', '1')


def run(x, groups, scale, shift, act, dy, accumulate=False):
    from stmi import ops
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, act=act, eps=B.EPS)
    dscale, dshift = torch.zeros((2, x.shape[3]), device=x.device) if accumulate else torch.full((2, x.shape[3]), 7.0, device=x.device)
    kw = {} if accumulate else {'accumulate': False}
    dx = ops.group_norm_bwd(x, dy, groups, stats, scale, shift, dscale, dshift, act=act, **kw)
    return {'y': y, 'dx': dx, 'dshift': dshift, 'dscale': dscale}


def case(shape, dtype, act, cuda):
    *dims, groups = shape
    x, scale, shift, dy = (t.to(cuda) for t in B.data(dims, groups, dtype, sum(dims)))
    return x, groups, scale, shift, act, B.away_from_zero(x, groups, scale, shift, act, dy)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', B.SHAPES, ids=B.name)
def test_every_output_within_its_bound(cuda, shape, dtype, form):
    from stmi import ops
    act = [ops.ACT_SILU, ops.ACT_NONE, ops.ACT_SIGMOID, ops.ACT_RELU][(shape[1] + shape[3]) % 4]
    args = case(shape, dtype, act, cuda)
    want, parts = B.results(*args)
    assert not B.faults(run(*args), want, B.bounds(parts), parts, dtype)


@pytest.mark.parametrize('act', ['RELU', 'SILU', 'NONE', 'SIGMOID'])
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', [(2, 16, 16, 128, 32), (2, 128, 128, 32, 8), (2, 61, 67, 35, 5)], ids=B.name)
def test_gradients_added_to_cleared_buffers(cuda, shape, dtype, act, form):
    """The default of group_norm_bwd: parameter gradients are added."""
    from stmi import ops
    args = case(shape, dtype, getattr(ops, 'ACT_' + act), cuda)
    want, parts = B.results(*args)
    assert not B.faults(run(*args, accumulate=True), want, B.bounds(parts), parts, dtype)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', [(2, 16, 16, 512, 32), (2, 17, 23, 32, 8), (3, 64, 64, 64, 32), (2, 45, 45, 16, 2), (2, 37, 30, 72, 3)], ids=B.name)
def test_the_two_forms_agree(cuda, shape, dtype, monkeypatch):
    """One block per group, and slices: each is within the bounds of the formula, so they are within twice those of each other
    (and two roundings of a stored value)."""
    from stmi import ops
    args = case(shape, dtype, ops.ACT_SILU, cuda)
    bound = B.bounds(B.results(*args)[1])
    a = run(*args)
    monkeypatch.setenv('STMI_NO_GN_UNITS', '1')
    b = run(*args)
    for k in a:
        h = 2 * B.HALF[dtype if k in ('y', 'dx') else torch.float32]
        d, size = (a[k].double() - b[k].double()).abs(), torch.maximum(a[k].double().abs(), b[k].double().abs())
        assert (d <= h * size + 2.02 * bound[k].reshape(d.shape)).all(), k
