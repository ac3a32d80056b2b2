"""Group norm with an activation (forward, backward) against the formula in 64 bits.

Tolerances, before any run.  u = 2^-24 is half a step of fp32; inputs are taken as the kernel sees them (rounded to the
tensor's type), so only the kernel's own roundings count.
  * A sum of k terms in fp32, whatever its order, is off by at most about (32 + 2 sqrt(k)) u of the sum of the terms'
    magnitudes: every partial sum rounds by u, the roundings are independent (standard deviation below u sqrt(k) / 3 of
    that magnitude even for one running sum), 2 sqrt(k) is six of them; 32 covers the merges and short fixed chains.
  * With M values a group, mean and variance inherit E = (64 + 2 sqrt(M)) u (1 + max|x| rstd): the mean is off by
    that many u of max|x|, which is max|x| rstd in units of xhat; the roundings of rstd (sum, division, square root),
    of scale * rstd, of the activation's exponential (its argument, at most 2^4 here, rounds by u, so exp by 16 u) and
    its reciprocal come to less than 64 u of max(1, |z|).
  * z is then off by at most E * (|scale| max|xhat| + max|z| + 1); no activation is steeper than 1.1.
  * g = dy act'(z): act' has a slope below 0.6, so g is off by |dy| (0.6 dz + 64 u).
  * dx = rstd (scale g - m1 - xhat m2): each of the three terms is a product of quantities with the errors above.
  * An output of bf16 rounds once more, by at most finfo(bf16).eps / 2 = 2^-8 of its value.
The ReLU's derivative jumps at z = 0: there dy is zero where |z| is below what z may be off by.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']
EPS = 1e-3


def data(shape, dtype, seed, mean=1.0, dev=1.0):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = torch.randn(shape, generator=g) * (0.5 + torch.randn(c, generator=g).abs()) * dev + torch.randn(c, generator=g) * mean
    scale, shift = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    return x.to(dtype), scale, shift, torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)


def act64(z, act):
    from stmi import ops
    s = 1.0 / (1.0 + torch.exp(-z))
    if act == ops.ACT_RELU:
        return z.clamp_min(0.0), (z > 0).double()
    if act == ops.ACT_SIGMOID:
        return s, s * (1 - s)
    if act == ops.ACT_SILU:
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def formula(x, groups, scale, shift, act, residual=None, dy=None, eps=EPS):
    """Everything in 64 bits, and how far z may be off."""
    n, h, w, c = x.shape
    D, M = c // groups, h * w * (c // groups)
    x = x.double().reshape(n, h * w, groups, D)
    scale, shift = scale.double().reshape(groups, D), shift.double().reshape(groups, D)
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xhat = (x - mean) * rstd
    z = xhat * scale + shift
    E = (64 + 2 * M ** 0.5) * U * (1 + (x.abs() * rstd).max().item())
    dz = E * (scale.abs().max().item() * xhat.abs().max().item() + z.abs().max().item() + 1)
    y, grad = act64(z, act)
    out = {'mean': mean.reshape(n, groups), 'rstd': rstd.reshape(n, groups), 'z': z.reshape(n, h, w, c), 'dz': dz, 'E': E,
           'y': y.reshape(n, h, w, c)}
    if residual is not None:
        out['y'] = out['y'] + residual.double()
    if dy is not None:
        dy = dy.double().reshape(x.shape)
        g = dy * grad
        m1, m2 = (g * scale).mean((1, 3), keepdim=True), (g * scale * xhat).mean((1, 3), keepdim=True)
        dx = rstd * (g * scale - m1 - xhat * m2)
        xm, sm, rm = xhat.abs().max().item() + 1, scale.abs().max().item(), rstd.max().item()
        dg = dy.abs() * (0.6 * dz + 64 * U)             # of g, element by element
        k = (32 + 2 * (n * h * w) ** 0.5) * U
        big = dy.abs().max().item() * sm * xm
        out.update(dx=dx.reshape(n, h, w, c), dshift=g.sum((0, 1)).reshape(-1), dscale=(g * xhat).sum((0, 1)).reshape(-1))
        # terms of dx: scale g (dg), m1, m2 (sums over the group of the same errors), xhat (E)
        out['dx_tol'] = rm * xm * (2 * dg.max().item() * sm * xm + 3 * E * big * xm)
        out['dshift_tol'] = (dg.sum((0, 1)) + k * g.abs().sum((0, 1))).max().item()
        out['dscale_tol'] = ((dg * xm).sum((0, 1)) + (k + 2 * E) * (g.abs() * xm).sum((0, 1))).max().item()
    return out


def near(got, want, tol, dtype=torch.float32):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    bad = (got - want).abs() > HALF[dtype] * want.abs() + 1.01 * tol
    bad |= ~torch.isfinite(got)
    assert not bad.any(), (int(bad.sum()), (got - want).abs().max().item(), tol)


SHAPES = [  # n, h, w, c, groups
    (1, 1, 1, 8, 2), (1, 1, 1, 1, 1), (2, 1, 1, 512, 32), (3, 1, 7, 3, 1), (1, 5, 3, 3, 3),
    (2, 16, 16, 512, 32), (2, 17, 23, 32, 8), (1, 64, 48, 128, 32), (2, 33, 31, 64, 64), (1, 40, 41, 64, 1),
    (2, 13, 27, 35, 5), (1, 19, 21, 101, 101), (1, 9, 11, 257, 1), (2, 7, 5, 1000, 8), (1, 3, 5, 2040, 8),
    (1, 2, 3, 4096, 32), (1, 3, 3, 4094, 2), (1, 2, 2, 4093, 1), (1, 40, 50, 4096, 4096), (2, 30, 31, 4095, 4095), (5, 6, 7, 24, 12), (2, 50, 40, 16, 16), (17, 3, 3, 96, 3),
    (1, 200, 150, 12, 3), (3, 45, 67, 20, 2), (1, 130, 110, 256, 32),
    # one block per group: full and over-full registers, columns that do not divide the block
    (3, 64, 64, 64, 32), (3, 32, 32, 48, 2), (2, 37, 30, 72, 3), (1, 63, 43, 120, 5), (1, 65, 64, 64, 16), (9, 1, 2, 64, 64),
    (1, 8, 8, 1024, 2), (2, 45, 45, 16, 2),
    # partials folded by a launch of their own: many groups, a large sample
    (1, 200, 200, 128, 128), (1, 513, 520, 64, 32),
]


@pytest.fixture(params=['chosen', 'slices'])
def form(request, monkeypatch):
    """The form the library chooses (small samples: one block per group), and the one that cuts samples into slices."""
    if request.param == 'slices':
        monkeypatch.setenv('STMI_NO_GN_UNITS', '1')


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_forward_and_backward(cuda, shape, dtype, form):
    from stmi import ops
    *dims, groups = shape
    act = [ops.ACT_SILU, ops.ACT_NONE, ops.ACT_SIGMOID, ops.ACT_RELU][(dims[1] + dims[3]) % 4]
    x, scale, shift, dy, _ = data(dims, dtype, sum(dims))
    if act == ops.ACT_RELU:
        f = formula(x, groups, scale, shift, act)
        dy = torch.where(f['z'].abs() < 4 * f['dz'], torch.zeros_like(dy), dy)
    f = formula(x, groups, scale, shift, act, dy=dy)
    dev = [t.to(cuda) for t in (x, scale, shift, dy)]
    y, stats = ops.group_norm_fwd(dev[0], groups, dev[1], dev[2], act=act, eps=EPS)
    near(y, f['y'], 1.1 * f['dz'], dtype)
    near(stats[..., 0] * f['rstd'].float().to(cuda), f['mean'] * f['rstd'].float().double(), f['E'])
    near(stats[..., 1], f['rstd'], f['E'] * f['rstd'].max().item())
    dscale, dshift = torch.full((2, dims[3]), 7.0, device=cuda)
    dx = ops.group_norm_bwd(dev[0], dev[3], groups, stats, dev[1], dev[2], dscale, dshift, act=act, accumulate=False)
    near(dx, f['dx'], f['dx_tol'], dtype)
    near(dshift, f['dshift'], f['dshift_tol'])
    near(dscale, f['dscale'], f['dscale_tol'])
    # added to what the buffers hold: one more rounding
    before = dscale.clone(), dshift.clone()
    dx2 = ops.group_norm_bwd(dev[0], dev[3], groups, stats, dev[1], dev[2], dscale, dshift, act=act)
    assert torch.equal(dx2, dx)
    assert torch.equal(dscale, before[0] + before[0]) and torch.equal(dshift, before[1] + before[1])
    # without parameter gradients
    assert torch.equal(ops.group_norm_bwd(dev[0], dev[3], groups, stats, dev[1], dev[2], None, None, act=act), dx)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('act', ['NONE', 'RELU', 'SIGMOID', 'SILU'])
@pytest.mark.parametrize('shape', [(2, 12, 20, 64, 16), (2, 70, 90, 32, 8), (1, 11, 13, 35, 7)], ids=lambda s: 'x'.join(map(str, s)))
def test_every_activation_with_residual(cuda, shape, act, dtype, form):
    from stmi import ops
    *dims, groups = shape
    act = getattr(ops, 'ACT_' + act)
    x, scale, shift, dy, residual = data(dims, dtype, 5)
    f = formula(x, groups, scale, shift, act)
    dy = torch.where(f['z'].abs() < 4 * f['dz'], torch.zeros_like(dy), dy)
    f = formula(x, groups, scale, shift, act, residual, dy)
    dev = [t.to(cuda) for t in (x, scale, shift, dy, residual)]
    y, stats = ops.group_norm_fwd(dev[0], groups, dev[1], dev[2], act=act, residual=dev[4], eps=EPS)
    near(y, f['y'], 1.1 * f['dz'] + U * f['y'].abs().max().item(), dtype)
    dscale, dshift = torch.zeros((2, dims[3]), device=cuda)
    dx = ops.group_norm_bwd(dev[0], dev[3], groups, stats, dev[1], dev[2], dscale, dshift, act=act)
    near(dx, f['dx'], f['dx_tol'], dtype)
    near(dshift, f['dshift'], f['dshift_tol'])
    near(dscale, f['dscale'], f['dscale_tol'])


def test_gradient_against_differences(cuda):
    """The loss sum(w y) moved along a random direction of (x, scale, shift): its central difference, taken with the
    formula in 64 bits, is the gradients' product with the direction (truncation h^2 = 1e-8 of the third derivative)."""
    from stmi import ops
    shape, groups = (2, 9, 11, 24), 6
    x, scale, shift, w, d = data(shape, torch.float32, 11)
    ds, dh = torch.randn(24, generator=torch.Generator().manual_seed(1)), torch.randn(24, generator=torch.Generator().manual_seed(2))
    h = 1e-4
    loss = lambda t: (formula(x.double() + t * d, groups, scale.double() + t * ds, shift.double() + t * dh, ops.ACT_SILU)['y'] * w.double()).sum().item()  # noqa: E731
    want = (loss(h) - loss(-h)) / (2 * h)
    dev = [t.to(cuda) for t in (x, scale, shift, w)]
    _, stats = ops.group_norm_fwd(dev[0], groups, dev[1], dev[2], act=ops.ACT_SILU, eps=EPS)
    gs, gh = torch.zeros((2, 24), device=cuda)
    dx = ops.group_norm_bwd(dev[0], dev[3], groups, stats, dev[1], dev[2], gs, gh, act=ops.ACT_SILU)
    terms = [dx.double().cpu() * d, gs.double().cpu() * ds, gh.double().cpu() * dh]
    size = sum(t.abs().sum().item() for t in terms)
    assert abs(sum(t.sum().item() for t in terms) - want) <= 1e-5 * size


def test_groups_equal_to_channels_is_the_instance_norm(cuda):
    from stmi import ops
    x, scale, shift, dy, _ = (t.to(cuda) for t in data((2, 24, 20, 32), torch.float32, 3))
    f = formula(x.cpu(), 32, scale.cpu(), shift.cpu(), ops.ACT_RELU)
    y, stats = ops.group_norm_fwd(x, 32, scale, shift, act=ops.ACT_RELU)
    y_in, stats_in = ops.instance_norm_fwd(x, scale, shift, act=ops.ACT_RELU)
    assert (y - y_in).abs().max().item() <= 2.2 * f['dz']
    assert stats.shape == stats_in.shape and (stats - stats_in).abs().max().item() <= 4 * f['E'] * stats_in.abs().max().item()


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('mean,dev', [(300.0, 1.0), (0.0, 1e-4), (0.0, 1e6)], ids=['mean', 'small', 'large'])
@pytest.mark.parametrize('shape', [(2, 16, 16, 64, 8), (1, 96, 100, 64, 8)], ids=lambda s: 'x'.join(map(str, s)))
def test_means_and_deviations_of_other_sizes(cuda, shape, mean, dev, dtype, form):
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, _, _ = data(dims, dtype, 8, mean, dev)
    f = formula(x, groups, scale, shift, ops.ACT_SIGMOID)
    y, _ = ops.group_norm_fwd(x.to(cuda), groups, scale.to(cuda), shift.to(cuda), act=ops.ACT_SIGMOID, eps=EPS)
    near(y, f['y'], 1.1 * f['dz'], dtype)


@pytest.mark.parametrize('where', ['first', 'last', 'middle'])
@pytest.mark.parametrize('shape', [(1, 16, 16, 64, 8), (1, 128, 128, 32, 4)], ids=lambda s: 'x'.join(map(str, s)))
def test_one_far_value(cuda, shape, where, form):
    """One value 1e5 deviations away, at a place a shifted sum might take as its shift."""
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, _, _ = data(dims, torch.float32, 9)
    at = {'first': 0, 'last': dims[1] * dims[2] - 1, 'middle': dims[1] * dims[2] // 2}[where]
    x.view(-1, dims[3])[at, 3] = 1e5
    f = formula(x, groups, scale, shift, ops.ACT_NONE)
    y, stats = ops.group_norm_fwd(x.to(cuda), groups, scale.to(cuda), shift.to(cuda), eps=EPS)
    near(stats[..., 1], f['rstd'], (64 + 2 * (dims[1] * dims[2] * dims[3] / groups) ** 0.5) * U * 8 * f['rstd'].max().item())
    near(y, f['y'], f['dz'])


@pytest.mark.parametrize('shape', [(3, 8, 8, 64, 8), (3, 72, 80, 32, 4), (2, 9, 7, 35, 5)], ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')], ids=['nan', 'inf', '-inf'])
def test_not_finite_values_stay_in_their_group(cuda, shape, bad, form):
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, dy, _ = data(dims, torch.bfloat16, 4)
    x, scale, shift, dy = (t.to(cuda) for t in (x, scale, shift, dy))
    D = dims[3] // groups
    for act in (ops.ACT_NONE, ops.ACT_RELU, ops.ACT_SIGMOID, ops.ACT_SILU):
        clean, st = ops.group_norm_fwd(x, groups, scale, shift, act=act)
        clean_dx = ops.group_norm_bwd(x, dy, groups, st, scale, shift, None, None, act=act)
        dirty = x.clone()
        dirty[1, 3, 2, 2 * D] = bad
        y, st = ops.group_norm_fwd(dirty, groups, scale, shift, act=act)
        dx = ops.group_norm_bwd(dirty, dy, groups, st, scale, shift, None, None, act=act)
        hit = torch.zeros(dims, dtype=torch.bool, device=cuda)
        hit[1, :, :, 2 * D:3 * D] = True
        for got, want in ((y, clean), (dx, clean_dx)):
            assert torch.isnan(got[hit]).all()
            assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('hw', [(4, 4), (90, 100)], ids=['small', 'large'])
def test_constant_groups(cuda, hw, dtype, form):
    from stmi import ops
    x = torch.full((2,) + hw + (32,), 3.3, dtype=dtype, device=cuda)
    scale, shift = torch.ones(32, device=cuda), torch.full((32,), 0.5, device=cuda)
    y, stats = ops.group_norm_fwd(x, 4, scale, shift, eps=EPS)
    # the mean of equal values rounds by at most (32 + 2 sqrt(M)) u of them, the variance is the square of that at most
    M = hw[0] * hw[1] * 8
    e = (32 + 2 * M ** 0.5) * U * 3.3 / EPS ** 0.5
    near(y, torch.full(x.shape, 0.5), 4 * e, dtype)
    dx = ops.group_norm_bwd(x, torch.ones_like(x), 4, stats, scale, shift, None, None)
    near(dx, torch.zeros(x.shape), 8 * (64 + 2 * M ** 0.5) * U / EPS ** 0.5, dtype)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', [(5, 16, 16, 128, 32), (3, 120, 130, 32, 8), (3, 11, 13, 35, 5), (3, 45, 61, 35, 5)], ids=lambda s: 'x'.join(map(str, s)))
def test_a_sample_does_not_depend_on_its_batch_and_bits_repeat(cuda, shape, dtype, form):
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, dy, _ = (t.to(cuda) for t in data(dims, dtype, 6))
    run = lambda a, b: (lambda y, st: (y, st, ops.group_norm_bwd(a, b, groups, st, scale, shift, None, None, act=ops.ACT_SILU)))(  # noqa: E731
        *ops.group_norm_fwd(a, groups, scale, shift, act=ops.ACT_SILU))
    whole = run(x, dy)
    for got, want in zip(run(x, dy), whole):
        assert torch.equal(got, want)
    for i in range(dims[0]):
        for got, want in zip(run(x[i:i + 1].clone(), dy[i:i + 1].clone()), whole):
            assert torch.equal(got[0], want[i])


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape', [(2, 16, 16, 64, 8), (2, 110, 100, 32, 8), (2, 13, 9, 35, 5)], ids=lambda s: 'x'.join(map(str, s)))
def test_places(cuda, shape, dtype, form):
    """Outputs in the inputs' own memory, and tensors at any element of a larger buffer (the values around stay)."""
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, dy, res = (t.to(cuda) for t in data(dims, dtype, 12))
    f = formula(x.cpu(), groups, scale.cpu(), shift.cpu(), ops.ACT_SILU, res.cpu(), dy.cpu())
    y, st = ops.group_norm_fwd(x, groups, scale, shift, act=ops.ACT_SILU, residual=res)
    dx = ops.group_norm_bwd(x, dy, groups, st, scale, shift, None, None, act=ops.ACT_SILU)
    a = x.clone()
    assert ops.group_norm_fwd(a, groups, scale, shift, act=ops.ACT_SILU, residual=res, out=a)[0] is a and torch.equal(a, y)
    b = res.clone()
    ops.group_norm_fwd(x, groups, scale, shift, act=ops.ACT_SILU, residual=b, out=b)
    assert torch.equal(b, y)
    for which in (0, 1):
        ins = [x.clone(), dy.clone()]
        ops.group_norm_bwd(ins[0], ins[1], groups, st, scale, shift, None, None, act=ops.ACT_SILU, out=ins[which])
        assert torch.equal(ins[which], dx)

    def at(t, k):
        buf = torch.full((t.numel() + 32,), 2.0, dtype=t.dtype, device=cuda)
        view = buf[k:k + t.numel()].view(t.shape)
        view.copy_(t)
        return buf, view

    for places in ((1, 1, 1, 1), (0, 0, 3, 0), (4, 4, 4, 4), (1, 2, 5, 7)):
        (_, xv), (_, rv), (ybuf, yv), (_, dyv) = (at(t, k) for t, k in zip((x, res, torch.zeros_like(x), dy), places))
        ops.group_norm_fwd(xv, groups, scale, shift, act=ops.ACT_SILU, residual=rv, out=yv)
        near(yv, f['y'], 1.1 * f['dz'] + U * f['y'].abs().max().item(), dtype)
        assert torch.equal(yv, y)           # a sample's bits do not depend on its place
        k, m = places[2], x.numel()
        assert (ybuf[:k] == 2).all() and (ybuf[k + m:] == 2).all()
        dxbuf, dxv = at(x, places[2])
        gs, gh = torch.zeros((2, dims[3]), device=cuda)
        ops.group_norm_bwd(xv, dyv, groups, st, scale, shift, gs, gh, act=ops.ACT_SILU, out=dxv)
        near(dxv, f['dx'], f['dx_tol'], dtype)
        assert torch.equal(dxv, dx)
        near(gs, f['dscale'], f['dscale_tol'])
        assert (dxbuf[:k] == 2).all() and (dxbuf[k + m:] == 2).all()


def test_more_than_2_to_31_elements(cuda):
    """One sample of more than 2^31 elements, twice: the second half of the tensor is a copy of the first."""
    from stmi import ops
    h, w, c, groups = 8195, 8200, 32, 4
    x = torch.empty((2, h, w, c), dtype=torch.bfloat16, device=cuda)
    assert x[0].numel() > 2 ** 31
    g = torch.Generator(device=cuda).manual_seed(1)
    for r in range(0, h, 1024):
        x[0, r:r + 1024] = torch.randn((min(1024, h - r), w, c), generator=g, device=cuda) + 0.01 * r
    x[1] = x[0]
    scale, shift = torch.linspace(0.5, 1.5, c, device=cuda), torch.linspace(-1, 1, c, device=cuda)
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, act=ops.ACT_SILU, eps=EPS)
    assert torch.equal(y[0], y[1]) and torch.equal(stats[0], stats[1])
    s1, s2 = torch.zeros(groups, dtype=torch.float64, device=cuda), torch.zeros(groups, dtype=torch.float64, device=cuda)
    for r in range(0, h, 512):
        v = x[0, r:r + 512].double().view(-1, groups, c // groups)
        s1 += v.sum((0, 2))
        s2 += (v ** 2).sum((0, 2))
    M = h * w * (c // groups)
    mean = s1 / M
    rstd = 1 / torch.sqrt(s2 / M - mean ** 2 + EPS)
    E = (64 + 2 * M ** 0.5) * U
    assert ((stats[0, :, 0].double() - mean).abs() <= E * 90).all() and ((stats[0, :, 1].double() / rstd - 1).abs() <= E * 4).all()
    dy = x          # any gradient will do: large and at hand
    dscale, dshift = torch.zeros((2, c), device=cuda)
    dx = ops.group_norm_bwd(x, dy, groups, stats, scale, shift, dscale, dshift, act=ops.ACT_NONE)
    assert torch.equal(dx[0], dx[1])
    want = torch.zeros(c, dtype=torch.float64, device=cuda)
    for r in range(0, h, 512):
        want += x[0, r:r + 512].double().sum((0, 1))
    assert ((dshift.double() / (2 * want) - 1).abs() <= (32 + 2 * (2 * h * w) ** 0.5) * U).all()
    # last pixels of the last sample, from the statistics
    m, rs = (stats[1, :, i].double().repeat_interleave(c // groups) for i in (0, 1))
    z = (x[1, -1, -3:].double() - m) * rs * scale.double() + shift.double()
    near(y[1, -1, -3:], (z / (1 + torch.exp(-z))).cpu(), 64 * U * (z.abs().max().item() + 1), torch.bfloat16)


@pytest.mark.parametrize('shape', [(2, 16, 16, 64, 8), (2, 120, 130, 32, 8)], ids=lambda s: 'x'.join(map(str, s)))
def test_captured_and_replayed_on_another_stream(cuda, shape):
    from stmi import ops
    *dims, groups = shape
    x, scale, shift, dy, _ = (t.to(cuda) for t in data(dims, torch.bfloat16, 2))

    def step(a, b):
        y, st = ops.group_norm_fwd(a, groups, scale, shift, act=ops.ACT_SILU)
        gs, gh = torch.empty((2, dims[3]), device=cuda)
        dx = ops.group_norm_bwd(a, b, groups, st, scale, shift, gs, gh, act=ops.ACT_SILU, accumulate=False)
        return y, dx, gs, gh

    step(x, dy)
    sx, sdy = x.clone(), dy.clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = step(sx, sdy)
    for seed in (21, 22, 23):
        nx, _, _, ndy, _ = (t.to(cuda) for t in data(dims, torch.bfloat16, seed))
        want = step(nx, ndy)
        sx.copy_(nx)
        sdy.copy_(ndy)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, step(x, dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('c,groups', [(3, 1), (8, 2)])
def test_more_samples_than_a_grid_dimension(cuda, c, groups):
    from stmi import ops
    n = 70001
    x, scale, shift, dy, _ = (t.to(cuda) for t in data((n, 2, 3, c), torch.float32, 40))
    f = formula(x.cpu(), groups, scale.cpu(), shift.cpu(), ops.ACT_SILU, dy=dy.cpu())
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, act=ops.ACT_SILU, eps=EPS)
    near(y, f['y'], 1.1 * f['dz'])
    gs, gh = torch.zeros((2, c), device=cuda)
    near(ops.group_norm_bwd(x, dy, groups, stats, scale, shift, gs, gh, act=ops.ACT_SILU), f['dx'], f['dx_tol'])
    near(gs, f['dscale'], f['dscale_tol'])
    near(gh, f['dshift'], f['dshift_tol'])


def test_more_threads_than_a_grid_dimension(cuda):
    """One block per group: 131075 samples of 512 groups are more than 2^32 threads.  Seven samples over and over: the batch
    gives the bits of the seven."""
    from stmi import ops
    times, c, groups = 18725, 4096, 512
    x, scale, shift, dy, _ = (t.to(cuda) for t in data((7, 1, 1, c), torch.bfloat16, 41))
    many = lambda t: t.repeat(times, 1, 1, 1)   # noqa: E731
    y, stats = ops.group_norm_fwd(x, groups, scale, shift, eps=EPS)
    dx = ops.group_norm_bwd(x, dy, groups, stats, scale, shift, None, None)
    yy, ss = ops.group_norm_fwd(many(x), groups, scale, shift, eps=EPS)
    assert torch.equal(yy, many(y)) and torch.equal(ss, stats.repeat(times, 1, 1))
    del yy
    gs, gh = torch.zeros((2, c), device=cuda)
    assert torch.equal(ops.group_norm_bwd(many(x), many(dy), groups, ss, scale, shift, gs, gh), many(dx))
    # a channel's terms are added in eight runs: each addition is off by 2^-24 of what the terms' sizes sum to
    mean, rstd = (stats[..., k].double().repeat_interleave(c // groups, 1) for k in (0, 1))
    d = dy.double().view(7, c)
    terms = d * (x.double().view(7, c) - mean) * rstd
    for got, t in ((gs, terms), (gh, d)):
        size = times * t.abs().sum(0)
        assert ((got.double() - times * t.sum(0)).abs() <= size * 2.0 ** -24 * (7 * times / 8 + 16)).all()


def test_empty_batch(cuda):
    from stmi import ops
    x = torch.empty((0, 4, 4, 8), device=cuda)
    scale, shift = torch.ones(8, device=cuda), torch.zeros(8, device=cuda)
    y, stats = ops.group_norm_fwd(x, 2, scale, shift)
    assert y.shape == x.shape and stats.shape == (0, 2, 2)
    gs, gh = torch.full((2, 8), 3.0, device=cuda)
    assert ops.group_norm_bwd(x, x, 2, stats, scale, shift, gs, gh).shape == x.shape
    assert (gs == 3).all() and (gh == 3).all()
    ops.group_norm_bwd(x, x, 2, stats, scale, shift, gs, gh, accumulate=False)
    assert (gs == 0).all() and (gh == 0).all()


def test_parameter_gradients_in_one_place_are_refused(cuda):
    from stmi import ops
    x = torch.zeros((2, 4, 4, 8), device=cuda)
    s, both = torch.ones(8, device=cuda), torch.zeros(16, device=cuda)
    y, stats = ops.group_norm_fwd(x, 2, s, s)
    for gs, gh in ((both[:8], both[:8]), (both[:8], both[4:12]), (both[4:12], both[:8])):
        with pytest.raises(ValueError, match='overlap'):
            ops.group_norm_bwd(x, x, 2, stats, s, s, gs, gh)
    ops.group_norm_bwd(x, x, 2, stats, s, s, both[8:], both[:8])   # neighbours are fine


def test_refusals(cuda):
    from stmi import lib, ops
    x = torch.zeros((2, 4, 4, 8), device=cuda)
    s = torch.ones(8, device=cuda)
    for groups in (3, 0, -1, 16):
        with pytest.raises((lib.StmiError, RuntimeError)):
            ops.group_norm_fwd(x, groups, s, s)
    with pytest.raises(lib.StmiError, match='bad activation'):
        ops.group_norm_fwd(x, 2, s, s, act=4)
    with pytest.raises(lib.StmiError, match='channels'):
        ops.group_norm_fwd(torch.zeros((1, 1, 1, 4097), device=cuda), 1, torch.ones(4097, device=cuda), torch.ones(4097, device=cuda))
    with pytest.raises(TypeError):
        ops.group_norm_fwd(x.half(), 2, s, s)
    with pytest.raises(TypeError):
        ops.group_norm_fwd(x, 2, s.double(), s)
    with pytest.raises(ValueError, match='contiguous'):
        ops.group_norm_fwd(x.permute(0, 2, 1, 3), 2, s, s)
    with pytest.raises(ValueError, match='shape'):
        ops.group_norm_fwd(x, 2, s[:4], s)
    with pytest.raises(ValueError, match='shape'):
        ops.group_norm_fwd(x, 2, s, s, residual=x[:1])
    buf = torch.zeros(x.numel() + 8, device=cuda)
    with pytest.raises(ValueError, match='overlaps'):
        ops.group_norm_fwd(buf[:-8].view(x.shape), 2, s, s, out=buf[8:].view(x.shape))
    with pytest.raises(ValueError, match='ws'):
        ops.group_norm_fwd(torch.zeros((1, 256, 256, 8), device=cuda), 2, s, s, ws=torch.empty(0, device=cuda))
    y, stats = ops.group_norm_fwd(x, 2, s, s)
    with pytest.raises(ValueError, match='together'):
        ops.group_norm_bwd(x, x, 2, stats, s, s, s.clone(), None)
    with pytest.raises(ValueError, match='shape'):
        ops.group_norm_bwd(x, x, 4, stats, s, s, None, None)
    with pytest.raises(lib.StmiError, match='no CPU fallback'):
        ops.group_norm_fwd(x.cpu(), 2, s, s)
    # the other operators do not take the new activation
    with pytest.raises(lib.StmiError):
        ops.activation(x, ops.ACT_SILU)
    with pytest.raises(lib.StmiError):
        ops.instance_norm_fwd(x, s, s, act=ops.ACT_SILU)
