"""Clipping and the clipped Adam where norms are very large."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('max_norm', [1.0, 1e-6, 1e-30, 3e-20])
def test_clipping_of_gradients_near_the_largest_number(cuda, dtype, max_norm):
    """norm / max_norm beyond fp32's range: out = g * factor in two products, at most 3 u (bf16: and 2^-8) of its value;
    2^-133: results below the smallest normal number round by that number's step."""
    from stmi import ops
    gen = torch.Generator().manual_seed(0)
    t = ((torch.rand(3001, generator=gen) + 0.5) * 2e38 * (torch.randint(0, 2, (3001,), generator=gen) * 2 - 1)).to(dtype)
    want_norm = t.double().norm().item()
    assert want_norm > 3.5e38 and want_norm < math.inf
    max_norm = float(torch.tensor(max_norm))
    want = t.double() * (max_norm / want_norm)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    src, out = t.to(cuda), torch.empty(3001, dtype=dtype, device=cuda)
    norm = ops.GradList([src], [out]).clip(max_norm)
    assert torch.isinf(norm).all()           # beyond fp32
    assert ((out.double().cpu() - want).abs() <= (half + 3 * U) * want.abs() + 2.0 ** -133).all()
    ops.GradList([src]).clip(max_norm)
    assert torch.equal(src, out)


@pytest.mark.parametrize('grad_scale,max_norm', [(1.0, 1.0), (0.125, 1e-3), (1e-30, 1e-6), (0.3, 1e-6)])
def test_adam_of_gradients_near_the_largest_number(cuda, grad_scale, max_norm):
    """m = (1 - b1) g': g' = g * grad_scale * factor rounds three times at most, the rate and the product once each; v squares
    it."""
    from stmi import ops
    gen = torch.Generator().manual_seed(1)
    g = (torch.rand(4099, generator=gen) + 0.5) * 2e38
    s = float(torch.tensor(grad_scale))
    norm, max_norm = g.double().norm().item() * s, float(torch.tensor(max_norm))
    want = g.double() * s * min(1.0, max_norm / norm)
    g = g.to(cuda)
    p, m, v = torch.zeros((3, 4099), device=cuda)
    lst = ops.GradList([g])
    lst.sum_squares()
    ops.adam_tf1(p, g, m, v, 1e-3, grad_scale=s, t=1, clip=lst, max_norm=max_norm)
    c1, c2 = 1 - 0.9, 1 - 0.999
    assert ((m.double().cpu() - c1 * want).abs() <= 5 * U * c1 * want + 2.0 ** -133).all()
    assert ((v.double().cpu() - c2 * want ** 2).abs() <= 9 * U * c2 * want ** 2 + 2.0 ** -133).all()
