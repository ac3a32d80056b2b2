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
