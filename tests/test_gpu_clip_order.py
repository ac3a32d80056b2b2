"""The clipped update takes the norm that its list's calls left: without one, or after a clip() that overwrote the tensors,
it is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def state(cuda, n=5000):
    gen = torch.Generator().manual_seed(2)
    p, g, m, v = (torch.randn(n, generator=gen).to(cuda) for _ in range(4))
    return p, g, m, v.abs_()


def test_update_without_the_norm_of_its_gradients_is_refused(cuda):
    from stmi import ops
    p, g, m, v = state(cuda)
    before = [t.clone() for t in (p, g, m, v)]
    update = lambda lst: ops.adam_tf1(p, g, m, v, 1e-3, t=1, clip=lst, max_norm=1.0)   # noqa: E731
    lst = ops.GradList([g])
    with pytest.raises(ValueError, match='sum_squares'):
        update(lst)
    lst.norm()
    lst.clip(0.5)                   # in place: the norm was that of the tensors before
    before[1] = g.clone()
    with pytest.raises(ValueError, match='sum_squares'):
        update(lst)
    torch.cuda.synchronize()
    for a, b in zip((p, g, m, v), before):
        assert torch.equal(a, b)
    lst.sum_squares()
    update(lst)
    # g has the norm 0.5 < 1 now: not clipped again
    c1 = 1 - 0.9
    want = 0.9 * before[2].double() + c1 * before[1].double()
    size = 0.9 * before[2].double().abs() + c1 * before[1].double().abs()
    assert ((m.double() - want).abs() <= 4 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize('call', ['norm', 'clip', 'sum_squares'])
def test_every_call_that_leaves_the_tensors_norm_allows_updates(cuda, call):
    from stmi import ops
    p, g, m, v = state(cuda)
    ref = [t.clone() for t in (p, g, m, v)]
    lst = ops.GradList([g], [torch.empty_like(g)])
    {'norm': lst.norm, 'clip': lambda: lst.clip(0.1), 'sum_squares': lst.sum_squares}[call]()
    for sl in (slice(0, 2000), slice(2000, 5000)):      # slices share the norm
        ops.adam_tf1(p[sl], g[sl], m[sl], v[sl], 1e-3, t=2, clip=lst, max_norm=0.5)
    other = ops.GradList([ref[1]])
    other.sum_squares()
    ops.adam_tf1(*ref, 1e-3, t=2, clip=other, max_norm=0.5)
    for a, b in zip((p, m, v), (ref[0], ref[2], ref[3])):
        assert torch.equal(a, b)


def test_a_norm_that_was_captured_and_never_replayed_is_seen(cuda):
    from stmi import ops
    p, g, m, v = state(cuda)
    ops.GradList([g]).norm()
    lst = ops.GradList([g])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        lst.sum_squares()
    ops.adam_tf1(p, g, m, v, 1e-3, t=1, clip=lst, max_norm=1.0)
    assert torch.isnan(p).all() and torch.isnan(m).all() and torch.isnan(v).all()
    p, g2, m, v = state(cuda)
    assert torch.equal(g, g2)
    graph.replay()
    ops.adam_tf1(p, g, m, v, 1e-3, t=1, clip=lst, max_norm=1.0)
    assert torch.isfinite(p).all()


def test_a_new_list_never_clips_by_what_memory_held(cuda):
    """The C entry itself, on a list's fresh workspace: NaN, whatever the allocator's memory held."""
    from stmi import lib, ops
    p, g, m, v = state(cuda)
    for _ in range(4):
        torch.full((lib.GRAD_WS_DOUBLES,), 1e-12, dtype=torch.float64, device=cuda)
    lst = ops.GradList([g])
    lib.call('stmi_adam_tf1_clip', p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), g.numel(), 1e-3, 0.9, 0.999, 1e-8,
             1.0, lst._ws_place, lst._n, 1.0, None, None, 1, torch.cuda.current_stream().cuda_stream)
    assert torch.isnan(p).all()
