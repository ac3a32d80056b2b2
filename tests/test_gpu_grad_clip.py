"""The global gradient norm, clipping, and Adam with clipping against the formulas in 64 bits.

Tolerances, before any run (u = 2^-24, half a step of fp32).  Squares of fp32 and bf16 values are summed in double, where a
product rounds by 2^-53: the norm is off by its one rounding to fp32, u (2 u allowed).  The factor rounds once (u), its
product with a gradient once more (u, or 2^-8 to bf16): 3 u resp. 2^-8 + 3 u of an output's value.  Adam: m and v are sums
of two products whose four coefficients round to fp32 (the rates come in double), 8 u of the terms' magnitudes; p moves by lr_t m / (sqrt(v) + eps), off by 16 u of the
step's size, and rounds by u.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LENGTHS = [
    [1], [0], [3], [4], [8191], [8192], [8193], [100003], [1677638],
    [0, 1, 0, 2, 3, 5, 8, 13, 4096, 0, 77], [7] * 300, list(range(1, 200)), [8192 * 3, 1, 8192 * 2 + 1, 16384], [1] * 3000,
]


def make(lengths, kinds, device, seed=0, scale=1e-2, offset=0):
    """Tensors as slices of one flat buffer per type, `offset` elements into it."""
    g = torch.Generator().manual_seed(seed)
    out, flat = [], {}
    for k in (torch.float32, torch.bfloat16):
        n = sum(a for i, a in enumerate(lengths) if kinds[i % len(kinds)] == k)
        flat[k] = [(torch.randn(n + offset, generator=g) * scale).to(k).to(device), offset]
    for i, n in enumerate(lengths):
        f = flat[kinds[i % len(kinds)]]
        out.append(f[0][f[1]:f[1] + n])
        f[1] += n
    return out


def norm64(ts):
    return math.sqrt(sum(t.double().cpu().pow(2).sum().item() for t in ts))


def check_scaled(outs, ins, norm, max_norm):
    f = min(1.0, max_norm / norm) if norm > 0 else 1.0
    for o, t in zip(outs, ins):
        half = 2.0 ** -8 if t.dtype == torch.bfloat16 else 0.0
        want = t.double().cpu() * f
        # values below the smallest normal number round by that number's step
        assert ((o.double().cpu() - want).abs() <= (half + 3 * U) * want.abs() + 2.0 ** -133).all()


@pytest.mark.parametrize('kinds', [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16, torch.bfloat16)], ids=['f32', 'bf16', 'mixed'])
@pytest.mark.parametrize('offset', [0, 1, 3])
@pytest.mark.parametrize('lengths', LENGTHS, ids=lambda v: '%dx%d' % (len(v), max(v)))
def test_norm_and_clip(cuda, lengths, kinds, offset):
    from stmi import ops
    ts = make(lengths, kinds, cuda, 3, offset=offset)
    ref = [t.clone() for t in ts]
    want = norm64(ts)
    outs = [torch.full_like(t, 9) for t in ts]
    both = ops.GradList(ts, outs)
    norm = both.norm()
    assert norm.shape == (1,) and abs(norm.item() - want) <= 2 * U * want
    for max_norm in (0.25 * want or 1.0, 4 * want or 1.0):
        assert torch.equal(both.clip(max_norm), norm)
        check_scaled(outs, ref, want, max_norm)
        if max_norm >= want:
            for o, t in zip(outs, ref):
                assert torch.equal(o, t)            # the factor is exactly 1
    for t, r in zip(ts, ref):
        assert torch.equal(t, r)
    own = ops.GradList(ts)
    assert torch.equal(own.clip(4 * want or 1.0), norm)
    for t, r in zip(ts, ref):
        assert torch.equal(t, r)
    if want:
        own.clip(0.25 * want)
        check_scaled(ts, ref, want, 0.25 * want)
        assert abs(own.norm().item() - 0.25 * want) <= (2.0 ** -8 + 4 * U) * want


def test_outputs_of_another_alignment_and_neighbours_stay(cuda):
    from stmi import ops
    for dt in (torch.float32, torch.bfloat16):
        for a, b in ((0, 1), (1, 0), (3, 5), (5, 3)):
            src, dst = torch.randn(50000, device=cuda).to(dt), torch.full((50000,), 9.0, device=cuda).to(dt)
            t, o = src[a:a + 20011], dst[b:b + 20011]
            want = norm64([t])
            ops.GradList([t], [o]).clip(1.0)
            check_scaled([o], [t], want, 1.0)
            assert (dst[:b] == 9).all() and (dst[b + 20011:] == 9).all()


def test_no_tensors(cuda):
    from stmi import ops
    for g in (ops.GradList([]), ops.GradList([torch.empty(0, device=cuda)])):
        assert g.norm().item() == 0 and g.clip(1.0).item() == 0


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')], ids=['nan', 'inf', '-inf'])
def test_a_norm_that_is_not_finite_makes_every_output_nan(cuda, bad):
    from stmi import ops
    ts = make([5, 9000, 300], (torch.float32, torch.bfloat16), cuda)
    outs = [torch.zeros_like(t) for t in ts]
    ts[1][777] = bad
    norm = ops.GradList(ts, outs).clip(1.0)
    assert not torch.isfinite(norm).any() and all(torch.isnan(o).all() for o in outs)
    own = ops.GradList(ts)
    own.clip(1.0)
    assert all(torch.isnan(t).all() for t in ts)


@pytest.mark.parametrize('size', [1e30, 3e38, 1e-30, 1e-38])
def test_squares_neither_overflow_nor_vanish(cuda, size):
    from stmi import ops
    t = torch.full((1000,), size, device=cuda)
    want = norm64([t])
    got = ops.GradList([t], [torch.empty_like(t)]).norm().item()
    assert (math.isinf(got) if want > 3.4028235e38 else abs(got - want) <= 2 * U * want)
    # also where the norm itself is beyond fp32: the factor comes from the double
    out = torch.empty_like(t)
    ops.GradList([t], [out]).clip(1e-3 * size if size > 1 else size)
    check_scaled([out], [t], want, float(torch.tensor(1e-3 * size if size > 1 else size)))


def test_more_than_2_to_31_elements(cuda):
    from stmi import ops
    n = 2 ** 31 + 8195
    t = torch.ones(n, dtype=torch.bfloat16, device=cuda)
    t[-1] = 4096.0
    want = math.sqrt(n - 1 + 4096.0 ** 2)
    g = ops.GradList([t])
    assert abs(g.norm().item() - want) <= 2 * U * want
    g.clip(want / 2)
    assert (t[:-1] == 0.5).all() and t[-1] == 2048.0


def test_captured_and_replayed(cuda):
    from stmi import ops
    ts = make([4000, 77, 20000], (torch.float32, torch.bfloat16), cuda)
    outs = [torch.zeros_like(t) for t in ts]
    lst = ops.GradList(ts, outs)
    norm = torch.zeros(1, device=cuda)
    lst.clip(0.1, norm=norm)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        lst.clip(0.1, norm=norm)
    for seed in (4, 5, 6):
        for t, new in zip(ts, make([4000, 77, 20000], (torch.float32, torch.bfloat16), cuda, seed)):
            t.copy_(new)
        other = [torch.zeros_like(t) for t in ts]
        eager = ops.GradList(ts, other).clip(0.1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager) and all(torch.equal(a, b) for a, b in zip(outs, other))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lst.clip(0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, norm)


def adam64(p, g, m, v, lr, b1, b2, eps, scale, t):
    c1, c2 = 1 - b1, 1 - b2
    g = g.double().cpu() * scale
    m, v = m.double().cpu(), v.double().cpu()
    m2, v2 = b1 * m + c1 * g, b2 * v + c2 * g * g
    lr_t = lr * math.sqrt(1 - b2 ** t) / (1 - b1 ** t)
    step = lr_t * m2 / (v2.sqrt() + eps)
    return p.double().cpu() - step, m2, v2, step, (b1 * m).abs() + (c1 * g).abs()


@pytest.mark.parametrize('count', [1, 3, 4, 255, 4097, 100003, 1677638])
@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('rel', [0.25, 4.0], ids=['clipped', 'not clipped'])
def test_adam_with_clipping(cuda, count, offset, rel):
    from stmi import ops
    g_ = torch.Generator().manual_seed(count)
    bufs = [(torch.randn(count + offset, generator=g_) * s).to(cuda) for s in (0.1, 0.01, 0.003)]
    bufs.append((torch.randn(count + offset, generator=g_) * 0.01).square().to(cuda))
    p, g, m, v = (b[offset:] for b in bufs)
    scale = 0.125
    norm = norm64([g]) * scale
    max_norm = float(torch.tensor(rel * norm))
    want = adam64(p, g, m, v, 1e-3, 0.9, 0.999, 1e-8, scale * min(1.0, max_norm / norm), 7)
    heads = [b[:offset].clone() for b in bufs]
    lst = ops.GradList([g])
    out = torch.zeros(1, device=cuda)
    before = g.clone()
    step_dev = torch.full((1,), 6, dtype=torch.int32, device=cuda)
    lst.sum_squares()
    ops.adam_tf1(p, g, m, v, 1e-3, grad_scale=scale, step_dev=step_dev, clip=lst, max_norm=max_norm, norm=out)
    assert abs(out.item() - norm) <= 2 * U * norm and step_dev.item() == 7
    assert torch.equal(g, before) and all(torch.equal(b[:offset], h) for b, h in zip(bufs, heads))
    assert ((m.double().cpu() - want[1]).abs() <= 8 * U * want[4]).all()
    assert ((v.double().cpu() - want[2]).abs() <= 8 * U * want[2]).all()
    # the step's m may cancel: its error is 8 u of the terms' magnitudes
    slack = 16 * U * want[3].abs() + 8 * U * want[4] * (want[3] / want[1]).abs() + U * want[0].abs() * 1.01
    assert ((p.double().cpu() - want[0]).abs() <= slack + 1e-30).all()


def test_adam_of_slices_shares_one_norm_and_not_finite_gradients_reach_everything(cuda):
    from stmi import ops
    make_ = lambda: [t.to(cuda) for t in (torch.randn(9000, generator=torch.Generator().manual_seed(i)) for i in range(4))]  # noqa: E731
    p, g, m, v = make_()
    v.abs_()
    ref = [t.clone() for t in (p, g, m, v)]
    lst = ops.GradList([g])
    lst.sum_squares()
    for sl in (slice(0, 4000), slice(4000, 9000)):
        ops.adam_tf1(p[sl], g[sl], m[sl], v[sl], 1e-3, t=3, clip=lst, max_norm=0.5)
    lst2 = ops.GradList([ref[1]])
    lst2.sum_squares()
    ops.adam_tf1(*ref, 1e-3, t=3, clip=lst2, max_norm=0.5)
    for a, b in zip((p, m, v), (ref[0], ref[2], ref[3])):
        assert torch.equal(a, b)
    g[17] = float('inf')
    lst.sum_squares()
    ops.adam_tf1(p, g, m, v, 1e-3, t=3, clip=lst, max_norm=0.5)
    assert torch.isnan(p).all() and torch.isnan(m).all() and torch.isnan(v).all()


def test_a_norm_layer_through_backward_clipping_and_update(cuda):
    """group norm -> convolution -> loss; the gradients of both layers clipped together and applied, against the same
    step in 64 bits (operators' own tolerances: 1e-3 of each tensor's maximum for the fp32 convolution kernels)."""
    from oracle import tf_ops as O
    from stmi import ops
    n, h, w, ci, co, groups = 2, 14, 10, 32, 64, 8
    gen = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=gen)   # noqa: E731
    x, wt, scale, shift, dy = rnd(n, h, w, ci), 0.1 * rnd(3, 3, ci, co), 1 + 0.1 * rnd(ci), 0.1 * rnd(ci), rnd(n, h, w, co)
    # 64 bits
    leaves = [t.double().requires_grad_(True) for t in (wt, scale, shift)]
    xg = x.double().view(n, h * w, groups, ci // groups)
    xhat = (xg - xg.mean((1, 3), keepdim=True)) / torch.sqrt(xg.var((1, 3), unbiased=False, keepdim=True) + 1e-3)
    z = xhat.reshape(n, h, w, ci) * leaves[1] + leaves[2]
    out = O.conv2d_same(z / (1 + torch.exp(-z)), leaves[0], 1)
    grads = torch.autograd.grad(out, leaves, dy.double())
    norm = math.sqrt(sum(g.pow(2).sum().item() for g in grads))
    max_norm = norm / 3
    # kernels: parameters and gradients in one flat buffer, as the executors keep them
    sizes = [t.numel() for t in (wt, scale, shift)]
    flat = torch.cat([t.reshape(-1) for t in (wt, scale, shift)]).to(cuda)
    flat_grad, m, v = torch.zeros_like(flat), torch.zeros_like(flat), torch.zeros_like(flat)
    cut = lambda f: [a.view(t.shape) for a, t in zip(f.split(sizes), (wt, scale, shift))]   # noqa: E731
    (dw, dscale, dshift), (wd, sd, hd) = cut(flat_grad), cut(flat)
    xd, dyd = x.to(cuda), dy.to(cuda)
    a, stats = ops.group_norm_fwd(xd, groups, sd, hd, act=ops.ACT_SILU)
    y = ops.conv2d_fwd(a, ops.pack_conv_weights(wd, ops.PACK_FWD, torch.float32), (3, 3, ci, co), 1)
    assert (y.double().cpu() - out.detach()).abs().max() <= 1e-3 * out.detach().abs().max()
    ops.conv2d_wgrad(a, dyd, (3, 3, ci, co), 1, out=dw)
    da = ops.conv2d_dgrad(dyd, ops.pack_conv_weights(wd, ops.PACK_DGRAD, torch.float32), (3, 3, ci, co), 1, (h, w))
    ops.group_norm_bwd(xd, da, groups, stats, sd, hd, dscale, dshift, act=ops.ACT_SILU, accumulate=False)
    for got, want in zip((dw, dscale, dshift), grads):
        assert (got.double().cpu() - want).abs().max() <= 1e-3 * want.abs().max()
    lst = ops.GradList([dw, dscale, dshift], cut(torch.empty_like(flat_grad)))
    assert abs(lst.clip(max_norm).item() - norm) <= 1e-3 * norm
    for got, want in zip(lst._keep[1], grads):
        assert (got.double().cpu() - want / 3).abs().max() <= 2e-3 * want.abs().max()
    lst.sum_squares()
    before = flat.clone()
    ops.adam_tf1(flat, flat_grad, m, v, 1e-3, t=1, clip=lst, max_norm=max_norm)
    assert abs(m.double().norm().item() / 0.1 - max_norm) <= 2e-3 * max_norm
    # Adam's first step moves every parameter by lr wherever its gradient is far above epsilon
    far = flat_grad.abs() > 1e-3
    assert ((flat - before)[far].abs() / 1e-3 - 1).abs().max() <= 1e-2


def test_trainer_clips_to_the_global_norm(cuda):
    import numpy as np
    from oracle import tf_ops as O
    from stmi.trainer import StyleTrainer
    rng = np.random.default_rng(0)
    batch = torch.tensor(rng.random((2, 32, 24, 3)).astype(np.float32), device=cuda)
    style = torch.tensor(rng.random((1, 30, 22, 3)).astype(np.float32))
    vggw, mean = O.synthetic_vgg_weights(seed=7, width_div=8, bias_scale=0.1), np.array([103.9, 116.8, 123.7], np.float32)

    def trainer(**kw):
        t = StyleTrainer(2, 32, 24, cuda, vggw, mean, 1e-2, 1e4, 1e8, dtype=torch.float32,
                         params=O.init_stylizer_params(seed=1), **kw)
        t.set_style_image(style)
        return t

    free, eager, graph = trainer(use_graph=False), trainer(use_graph=False, max_grad_norm=1.0), trainer(max_grad_norm=1.0)
    for t in (free, eager, graph):
        t.step(batch)
    g = free.net.flat_grad.double()
    norm = g.norm().item()
    assert norm > 2.0 and torch.equal(free.net.flat_grad, eager.net.flat_grad)
    assert abs(eager.grad_norm.item() - norm) <= 2 * U * norm
    # first step: m = (1 - b1) g'
    c1 = 1 - 0.9
    assert ((eager.m.double() - c1 * g / norm).abs() <= 8 * U * (c1 * g / norm).abs() + 2.0 ** -133).all()
    for _ in range(2):
        eager.step(batch)
        graph.step(batch)
    assert torch.equal(eager.net.flat, graph.net.flat) and torch.equal(eager.grad_norm, graph.grad_norm)
    with pytest.raises(ValueError, match='max_grad_norm'):
        trainer(max_grad_norm=0.0)


class TwoEqualRanks:
    """Gradient buckets of a group of two ranks with equal gradients: a bucket holds the sum once it has been waited for,
    and not before."""

    def __init__(self, flat, ranges):
        self.flat, self.ranges, self.pending, self.log = flat, list(ranges), set(), []
        self.replay_seconds, self.replays, self.steps = 0.0, 0, 0

    def reduce_bucket(self, i):
        self.pending.add(i)

    def wait_bucket(self, i):
        if i in self.pending:
            self.pending.remove(i)
            self.log.append(i)
            self.flat[slice(*self.ranges[i])].mul_(2.0)

    def wait(self):
        for i in sorted(self.pending):
            self.wait_bucket(i)


@pytest.mark.parametrize('use_graph', [False, True], ids=['eager', 'graph'])
def test_data_parallel_trainer_clips_the_mean_of_all_buckets(cuda, use_graph, monkeypatch):
    import numpy as np
    import torch.distributed as dist
    from oracle import tf_ops as O
    from stmi import trainer as T
    monkeypatch.setattr(dist, 'barrier', lambda group=None: None)
    rng = np.random.default_rng(1)
    batch = torch.tensor(rng.random((1, 32, 32, 3)).astype(np.float32), device=cuda)
    style = torch.tensor(rng.random((1, 32, 32, 3)).astype(np.float32))
    make = lambda **kw: T.StyleTrainer(1, 32, 32, cuda, O.synthetic_vgg_weights(seed=5, width_div=8), np.zeros(3, np.float32),   # noqa: E731
                                       1e3, 1.0, 10.0, params=O.init_stylizer_params(seed=3), max_grad_norm=0.5, **kw)
    one, two = make(use_graph=False), make(use_graph=use_graph)
    assert len(T.BWD_SEGMENTS) > 1
    two.world = 2
    two.buckets = TwoEqualRanks(two.net.flat_grad, [two.net.param_range(hi, lo) for hi, lo in T.BWD_SEGMENTS])
    for t in (one, two):
        t.set_style_image(style)
        for _ in range(2):
            t.step(batch)
    torch.cuda.synchronize()
    assert one.grad_norm.item() > 1.0
    # the mean of two equal gradients is the gradient: same norm, same update (doubling and halving are exact)
    assert torch.equal(one.grad_norm, two.grad_norm) and torch.equal(one.net.flat, two.net.flat)


def test_refusals(cuda):
    from stmi import lib, ops
    t = torch.zeros(100, device=cuda)
    with pytest.raises(TypeError):
        ops.GradList([t.double()])
    with pytest.raises(lib.StmiError, match='no CPU fallback'):
        ops.GradList([t.cpu()])
    with pytest.raises(ValueError, match='contiguous'):
        ops.GradList([t.view(10, 10).t()])
    with pytest.raises(ValueError, match='outputs'):
        ops.GradList([t], [])
    with pytest.raises(ValueError, match='shape'):
        ops.GradList([t], [t[:50]])
    with pytest.raises(TypeError):
        ops.GradList([t], [t.bfloat16()])
    with pytest.raises(ValueError, match='overlaps'):
        ops.GradList([t, t])
    lst = ops.GradList([t])
    for bad in (0.0, -1.0, float('inf'), float('nan')):
        with pytest.raises(lib.StmiError, match='max_norm'):
            lst.clip(bad)
        with pytest.raises(lib.StmiError, match='max_norm'):
            ops.adam_tf1(t, t.clone(), t.clone(), t.clone(), 1e-3, t=1, clip=lst, max_norm=bad)
    with pytest.raises(ValueError, match='shape'):
        lst.norm(out=torch.zeros(2, device=cuda))
    with pytest.raises(ValueError, match='together'):
        ops.adam_tf1(t, t.clone(), t.clone(), t.clone(), 1e-3, t=1, clip=lst)
    with pytest.raises(ValueError, match='together'):
        ops.adam_tf1(t, t.clone(), t.clone(), t.clone(), 1e-3, t=1, norm=t[:1])
