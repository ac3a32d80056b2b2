"""The bounds that the group norm's kernels are held to see what they are for: the results in 32 bits stay inside them, results
with a term, a slice or the last pixel missing do not.  Mistakes are planted in the formula, no GPU."""
import pytest
import torch

import group_norm_bounds as B

DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


def case(shape, dtype, act=None):
    from stmi import ops
    *dims, groups = shape
    act = [ops.ACT_SILU, ops.ACT_NONE, ops.ACT_SIGMOID, ops.ACT_RELU][(dims[1] + dims[3]) % 4] if act is None else act
    x, scale, shift, dy = B.data(dims, groups, dtype, sum(dims))
    args = (x, groups, scale, shift, act, B.away_from_zero(x, groups, scale, shift, act, dy))
    want, parts = B.results(*args)
    return args, want, parts, B.bounds(parts)


def stored(out, dtype):
    return {k: v.to(dtype if k in ('y', 'dx') else torch.float32) for k, v in out.items()}


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', B.SHAPES, ids=B.name)
def test_bounds_tell_right_from_wrong(shape, dtype):
    args, want, parts, bound = case(shape, dtype)
    n, P, G, D = parts['v'].shape
    seen = lambda out, *only: B.faults({k: v for k, v in stored(out, dtype).items() if not only or k in only}, want, bound, parts, dtype)   # noqa: E731
    assert not seen(want)
    assert not seen(B.results(*args, kind=torch.float32)[0])
    large = args[0].numel() > 1 << 21      # the mistakes that are hardest to see only: a pass takes seconds
    if not large:
        for kw in (dict(m1=False), dict(m2=False), dict(m1=False, m2=False)):
            assert seen(B.results(*args, **kw)[0], 'dx'), kw
        none = B.results(*args, eps=0.0)[0]
        assert seen(none, 'dx') and (dtype == torch.bfloat16 or seen(none, 'y'))
        for name in want:
            assert seen({name: torch.zeros_like(want[name])}), name
    # one of 512 slices (the most a sample is cut into), and the last pixel of few: left out of the sums
    lost = B.results(*args, lost=slice(0, -(-P // 512)))[0]
    assert seen(lost, 'dshift') and seen(lost, 'dscale')
    if dtype == torch.float32 or P * D <= 1 << 15:
        assert seen(lost, 'dx')
    if P <= 512:
        last = B.results(*args, lost=slice(P - 1, P))[0]
        assert seen(last, 'dx') and seen(last, 'dshift') and seen(last, 'dscale')


@pytest.mark.parametrize('act', ['NONE', 'RELU', 'SIGMOID', 'SILU'])
@pytest.mark.parametrize('shape', [(2, 5, 7, 12, 3), (1, 3, 2, 8, 8), (3, 4, 4, 6, 1)], ids=B.name)
def test_the_formula_is_the_derivative(shape, act):
    """dx, dscale and dshift of the formula against automatic differentiation of its y, in 64 bits, and against the central
    difference of sum(dy y) along a random direction: h^2 = 1e-8 of the third derivative, and 1e-16 / h of the sum."""
    from stmi import ops
    act = getattr(ops, 'ACT_' + act)
    *dims, groups = shape
    x, scale, shift, dy = (t.double() for t in B.data(dims, groups, torch.float32, 9))
    x = x * 3
    got, parts = B.results(x, groups, scale, shift, act, dy)
    leaves = [t.clone().requires_grad_(True) for t in (x, scale, shift)]
    want = torch.autograd.grad(B.results(leaves[0], groups, leaves[1], leaves[2], act, dy)[0]['y'], leaves, dy.reshape(got['y'].shape))
    for a, b in zip((got['dx'], got['dscale'], got['dshift']), want):
        assert (a.reshape(b.shape) - b).abs().max() <= 1e-12 * (1 + b.abs().max())
    h, gen = 1e-4, torch.Generator().manual_seed(1)
    assert act != ops.ACT_RELU or parts['z'].abs().min() > 10 * h      # no kink within the difference
    way = [torch.randn(t.shape, generator=gen).double() * 0.1 for t in (x, scale, shift)]
    loss = lambda t: (B.results(x + t * way[0], groups, scale + t * way[1], shift + t * way[2], act, dy)[0]['y'] * dy.reshape(got['y'].shape)).sum().item()   # noqa: E731
    terms = [a.reshape(b.shape) * b for a, b in zip((got['dx'], got['dscale'], got['dshift']), way)]
    assert abs((loss(h) - loss(-h)) / (2 * h) - sum(t.sum().item() for t in terms)) <= 1e-6 * sum(t.abs().sum().item() for t in terms)
