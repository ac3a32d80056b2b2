"""Group norm in 64 bits with a bound for every element: what fp32 kernels may be off by, derived from the formulas.

u = 2^-24 is half a step of fp32; inputs are taken as the kernel sees them.  All quantities belong to one group (one element)
of their own: no maxima over the tensor, so that a missing term shows where it acts.
  eps_M   a sum of M terms in fp32, in whatever order, is off by at most (64 + 2 sqrt(M)) u of the sum of the terms' sizes: every
          partial sum rounds by u of it at most, the roundings are independent (a standard deviation below u sqrt(M) / 3 even for
          one running sum, 2 sqrt(M) is six of them), 64 covers short fixed chains and merges.
  xhat    the mean is off by eps_M of the mean size of x, in units of the deviation d = eps_M (1 + mean|x| rstd); the variance is
          a sum of positive terms (and d^2, far below), its root halves the relative error: e_xhat = d + eps_M |xhat| + 4u |xhat|
  z       e_z = |scale| e_xhat + 4u (|scale xhat| + |shift|)
  y       no activation is steeper than 1.1; its exponential (an argument up to 2^4 rounds by u) and its reciprocal come to
          less than 64u (1 + |z|):  e_y = 1.1 e_z + 64u (1 + |z|)
  g       g = dy act'(z); act' is no steeper than 0.5 (SiLU), 0.1 (sigmoid), 0 (none; ReLU away from z = 0):
          e_g = |dy| (0.5 e_z + 64u (1 + |z|)) for the first two, 4u |g| for the others
  m1, m2  means of scale g and scale g xhat: the mean of their terms' errors, and eps_M of the mean size
  dx      rstd (|scale| e_g + e_m1 + |xhat| e_m2 + |m2| e_xhat + (eps_M + 16u) (|scale g| + |m1| + |xhat m2|))
  dshift  the sum of e_g and eps_nP sum|g|;  dscale: of e_g |xhat| + |g| e_xhat, and eps_nP sum|g xhat|
A stored value rounds by h = finfo / 2 of it once more.  In a sum of k stored values these roundings are independent and at most
h |v_i| each: they sum to no more than 8 h sqrt(sum v_i^2) (Hoeffding: missed once in 10^13), nor than h sum|v_i|.
"""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
EPS = 1e-3


def data(shape, groups, dtype, seed):
    """x with a deviation of 0.3 about channel means of 0.2 (eps = 1e-3 counts), dy with a mean and a part along xhat (so that
    both group terms of dx are of dx's own size)."""
    g = torch.Generator().manual_seed(seed)
    n, h, w, c = shape
    x = (torch.randn(shape, generator=g) * (0.2 + 0.1 * torch.rand(c, generator=g)) + 0.2 * torch.randn(c, generator=g)).to(dtype)
    scale, shift = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    v = x.float().view(n, h * w, groups, -1)
    xhat = (v - v.mean((1, 3), keepdim=True)) / (v.var((1, 3), unbiased=False, keepdim=True) + EPS).sqrt()
    dy = torch.randn(shape, generator=g) + 1.0 + 0.7 * xhat.view(shape)
    return x, scale, shift, dy.to(dtype)


def _act(z, act):
    from stmi import ops
    s = 1.0 / (1.0 + torch.exp(-z))
    if act == ops.ACT_RELU:
        return z.clamp_min(0.0), (z > 0).to(z.dtype), 0.0
    if act == ops.ACT_SIGMOID:
        return s, s * (1 - s), 0.1
    if act == ops.ACT_SILU:
        return z * s, s * (1 + z * (1 - s)), 0.5
    return z, torch.ones_like(z), 0.0


def results(x, groups, scale, shift, act, dy, eps=EPS, kind=torch.float64, m1=True, m2=True, lost=None):
    """The operator in elementary torch operations of type `kind`; m1, m2 False: without that term of dx; lost: pixels of every
    sample that are left out of the backward pass's sums."""
    n, h, w, c = x.shape
    cut = lambda t: t.to(kind).reshape(n, h * w, groups, c // groups)   # noqa: E731
    v, dv = cut(x), cut(dy)
    a, b = (t.to(kind).reshape(groups, -1) for t in (scale, shift))
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xhat = (v - mean) * rstd
    z = xhat * a + b
    y, grad, steep = _act(z, act)
    g = dv * grad
    kept = g if lost is None else g.clone()
    if lost is not None:
        kept[:, lost] = 0
    t1 = (kept * a).mean((1, 3), keepdim=True)
    t2 = (kept * a * xhat).mean((1, 3), keepdim=True)
    dx = rstd * (g * a - t1 * m1 - xhat * t2 * m2)
    out = {'y': y, 'dx': dx, 'dshift': kept.sum((0, 1)), 'dscale': (kept * xhat).sum((0, 1))}
    return out, dict(v=v, dy=dv, a=a, b=b, mean=mean, rstd=rstd, xhat=xhat, z=z, g=g, m1=t1, m2=t2, steep=steep)


def bounds(p):
    """{output: how far it may be off, element by element, before its own rounding} from the parts of results()."""
    n, P, _, D = p['v'].shape
    avg = lambda t: t.mean((1, 3), keepdim=True)   # noqa: E731
    eM, eN = ((64 + 2 * k ** 0.5) * U for k in (P * D, n * P))
    xhat, z, g, a = p['xhat'].abs(), p['z'].abs(), p['g'].abs(), p['a'].abs()
    ex = eM * (1 + avg(p['v'].abs()) * p['rstd']) + (eM + 4 * U) * xhat
    ez = a * ex + 4 * U * (a * xhat + p['b'].abs())
    eg = p['dy'].abs() * (0.5 * ez + 64 * U * (1 + z)) if p['steep'] else 4 * U * g
    e1 = avg(a * eg) + eM * avg(a * g)
    e2 = avg(a * (eg * xhat + g * ex)) + eM * avg(a * g * xhat)
    dx = p['rstd'] * (a * eg + e1 + xhat * e2 + p['m2'].abs() * ex + (eM + 16 * U) * (a * g + p['m1'].abs() + xhat * p['m2'].abs()))
    return {'y': 1.1 * ez + 64 * U * (1 + z), 'dx': dx, 'dshift': eg.sum((0, 1)) + eN * g.sum((0, 1)),
            'dscale': (eg * xhat + g * ex).sum((0, 1)) + eN * (g * xhat).sum((0, 1)), 'z': ez}


def away_from_zero(x, groups, scale, shift, act, dy):
    """dy without the places where the ReLU's derivative depends on z's roundings."""
    from stmi import ops
    if act != ops.ACT_RELU:
        return dy
    _, p = results(x, groups, scale, shift, act, dy)
    return torch.where((p['z'].abs() < 4 * bounds(p)['z']).reshape(dy.shape), torch.zeros_like(dy), dy)


def faults(got, want, bound, p, dtype):
    """What is out of bounds: a list of texts, empty if nothing is.  got: {name: tensor}, y and dx of type dtype."""
    bad = []
    for name, t in got.items():
        w, h = want[name], HALF[dtype if name in ('y', 'dx') else torch.float32]
        d = t.double().to(w.device).reshape(w.shape) - w
        over = d.abs() - (h * w.abs() + 1.01 * bound[name])
        if not bool((over <= 0).all()):          # NaN is over, too
            bad.append('%s: %d of %d elements, worst by %.3g' % (name, int((~(over <= 0)).sum()), d.numel(), over.max().item()))
        if name == 'dx':
            # along 1 and along xhat, group by group: where the two means act
            for k, q in (('1', torch.ones_like(w)), ('xhat', p['xhat'])):
                s, ww = (d * q).sum((1, 3)), (w * q)
                lim = 1.01 * (bound[name] * q.abs()).sum((1, 3)) + h * torch.minimum(8 * ww.square().sum((1, 3)).sqrt(), ww.abs().sum((1, 3)))
                if not bool((s.abs() <= lim).all()):
                    bad.append('dx along %s: %.3g times the bound' % (k, (s.abs() / lim).max().item()))
    return bad


SHAPES = [  # n, h, w, c, groups: one block per group, slices, tails, tiles of wide rows, folds by a launch of their own
    (1, 1, 7, 8, 2), (2, 16, 16, 512, 32), (2, 17, 23, 32, 8), (2, 33, 31, 64, 64), (2, 13, 27, 35, 5), (1, 19, 21, 101, 101),
    (1, 9, 11, 257, 1), (2, 7, 5, 1000, 8), (2, 12, 9, 513, 1), (1, 6, 5, 2052, 2), (1, 2, 3, 4096, 32), (1, 6, 7, 4093, 1), (1, 40, 50, 4096, 4096),
    (1, 20, 11, 4095, 4095), (5, 6, 7, 24, 12), (2, 50, 40, 16, 16), (3, 45, 67, 20, 2), (1, 130, 110, 256, 32), (3, 64, 64, 64, 32),
    (2, 37, 30, 72, 3), (1, 63, 43, 120, 5), (1, 65, 64, 64, 16), (2, 45, 45, 16, 2), (1, 200, 200, 128, 128), (4, 120, 130, 32, 8),
    (1, 513, 520, 64, 32),
]


def name(shape):
    return 'x'.join(map(str, shape))
