"""Host side of the group norm and the gradient list: refusals of the C-ABI, workspace sizes, the chunk table, and the
check for overlapping tensors.  No GPU."""
import ctypes

import pytest
import torch


def test_group_norm_arguments():
    from stmi import lib
    h = lib.load()
    ws = lambda *a: h.stmi_group_norm_ws_floats(*a, 0)   # noqa: E731
    assert ws(2, 256, 256, 64, 8, lib.F32) > 0 and ws(0, 8, 8, 64, 8, lib.BF16) == 0
    # one block per group: no workspace forward; a row of sums per sample backward, none for one sample
    assert ws(2, 8, 8, 64, 8, lib.BF16) == 0
    assert [h.stmi_group_norm_ws_floats(n, 8, 8, 64, 8, lib.BF16, 1) for n in (1, 3)] == [0, 3 * 2 * 64]
    assert h.stmi_group_norm_nhwc_fwd(1, None, 1, 1e-3, 1, 1, None, 1, 0, 2, 256, 256, 64, 8, 0, None) == -1
    for bad in ((2, 8, 8, 64, 7, 0), (2, 8, 8, 64, 0, 0), (2, 8, 8, 64, -8, 0), (2, 0, 8, 64, 8, 0), (2, 8, 0, 64, 8, 0),
                (-1, 8, 8, 64, 8, 0), (2, 8, 8, 0, 8, 0), (2, 8, 8, 64, 8, 2), (2, 8, 8, 4097, 1, 0), (1, 65536, 32768, 8, 1, 0)):
        assert ws(*bad) == -1, bad
        assert h.stmi_last_error()
    fwd = lambda act, *a: h.stmi_group_norm_nhwc_fwd(1, 1, 1, 1e-3, 1, 1, None, 1, act, *a, None)   # noqa: E731
    assert fwd(4, 2, 8, 8, 64, 8, 0) == -1 and b'activation' in h.stmi_last_error()
    assert fwd(-1, 2, 8, 8, 64, 8, 0) == -1
    assert fwd(0, 2, 8, 8, 64, 24, 0) == -1 and b'multiple' in h.stmi_last_error()
    assert fwd(0, 2, 8, 8, 64, 8, 5) == -1 and b'dtype' in h.stmi_last_error()
    for eps in (0.0, -1e-3, float('nan'), float('inf')):
        assert h.stmi_group_norm_nhwc_fwd(1, 1, 1, eps, 1, 1, None, 1, 0, 2, 8, 8, 64, 8, 0, None) == -1
        assert b'eps' in h.stmi_last_error()
    assert h.stmi_group_norm_nhwc_fwd(None, 1, 1, 1e-3, 1, 1, None, 1, 0, 2, 8, 8, 64, 8, 0, None) == -1
    assert h.stmi_group_norm_nhwc_fwd(None, None, None, 1e-3, None, None, None, None, 0, 0, 8, 8, 64, 8, 0, None) == 0   # empty batch
    bwd = lambda x, ds, dh: h.stmi_group_norm_nhwc_bwd(x, 1, 1, 1, 1, 1, ds, dh, 0, 1, 0, 2, 8, 8, 64, 8, 0, None)   # noqa: E731
    assert bwd(None, 1, 1) == -1 and bwd(1, 1, None) == -1 and bwd(1, None, 1) == -1


def fill(lengths, dtypes, src, dst):
    from stmi import lib
    h, n = lib.load(), len(lengths)
    counts = (ctypes.c_long * n)(*lengths)
    k = h.stmi_grad_list_chunks(counts, (ctypes.c_int * n)(*dtypes), n)
    table = (lib.GradChunk * max(k, 1))()
    rc = h.stmi_grad_list_fill((ctypes.c_void_p * n)(*src), (ctypes.c_void_p * n)(*dst), counts, (ctypes.c_int * n)(*dtypes), n, table)
    return rc, [(c.src, c.dst, c.count, c.dtype) for c in table[:k]]


def test_chunks_tile_every_tensor():
    lengths, dtypes = [0, 1, 8192, 8193, 100000, 2 ** 31 + 7], [0, 1, 0, 1, 1, 1]
    src = [i << 40 for i in range(1, 7)]
    dst = [(i << 40) + (1 << 36) for i in range(1, 7)]
    rc, table = fill(lengths, dtypes, src, dst)
    assert rc == 0
    got = iter(table)
    for n, dt, s, d in zip(lengths, dtypes, src, dst):
        size, at = 2 if dt else 4, 0
        while at < n:
            cs, cd, count, cdt = next(got)
            assert (cs, cd, cdt) == (s + at * size, d + at * size, dt) and 0 < count <= n - at
            at += count
    assert next(got, None) is None


def test_chunk_table_refusals():
    from stmi import lib
    h = lib.load()
    assert fill([4], [7], [16], [16])[0] == -1 and b'dtype' in h.stmi_last_error()
    assert fill([4], [0], [18], [16])[0] == -1 and b'aligned' in h.stmi_last_error()
    assert fill([4], [1], [16], [17])[0] == -1
    assert fill([4], [0], [None], [16])[0] == -1
    assert fill([0], [0], [None], [None]) == (0, [])
    assert h.stmi_grad_list_chunks((ctypes.c_long * 1)(-1), (ctypes.c_int * 1)(0), 1) == -1
    assert h.stmi_grad_clip(None, 3, 1, 1.0, None, None) == -1
    assert h.stmi_grad_norm(1, 3, 1, None, None) == -1
    assert h.stmi_grad_sum_squares(1, -1, 1, None) == -1
    for bad in (0.0, -2.0, float('inf'), float('nan')):
        assert h.stmi_grad_clip(1, 3, 1, bad, None, None) == -1 and b'max_norm' in h.stmi_last_error()
        assert h.stmi_adam_tf1_clip(1, 1, 1, 1, 8, 1e-3, .9, .999, 1e-8, 1.0, 1, 3, bad, None, None, 1, None) == -1
    assert h.stmi_adam_tf1_clip(1, 1, 1, 1, 8, 1e-3, .9, .999, 1e-8, 1.0, 1, 3, 1.0, None, None, 0, None) == -1
    assert h.stmi_adam_tf1_clip(1, 1, 1, 1, 8, 1e-3, .9, .999, 1e-8, 1.0, None, 3, 1.0, None, None, 1, None) == -1


def test_overlapping_outputs_are_refused():
    from stmi.ops import _chk_disjoint
    a, b, e = torch.zeros(100), torch.zeros(100), torch.zeros(0)
    ok = [([a, b], [a, b]), ([a, b], [b.clone(), a.clone()]), ([a[:50], a[50:]], [a[:50], a[50:]]), ([a, a], [b, b.clone()]),
          ([a[:60], a[40:]], [b[:60], b.clone()[40:]]), ([e, e], [e, e]), ([], []), ([a[:50], b], [a[50:], b])]
    bad = [([a, a], [a, a]), ([a, b], [b, a]), ([a], [b, ][:1] + []) if False else ([a, b], [a, a]), ([a[:50]], [a[1:51]]),
           ([a[:50], a[40:90]], [a[:50], b[:50]]), ([a, b], [b, b.clone()]), ([a[:60], a[40:]], [a[:60], a[40:]]),
           ([a, a[:1]], [a, b[:1]]), ([a, a[99:]], [b, a[99:]]), ([a, b[:1], b], [a, torch.zeros(1), b])]
    for ts, outs in ok:
        _chk_disjoint(ts, outs)
    for ts, outs in bad:
        with pytest.raises(ValueError, match='overlaps'):
            _chk_disjoint(ts, outs)
    for same in ([a, a], [a, a[:1]], [a, a[99:]], [b, a[:60], a[40:]]):
        with pytest.raises(ValueError, match='overlaps'):
            _chk_disjoint(same, same)
    pieces = [a[i:i + 1] for i in range(100)]
    _chk_disjoint(pieces[::-1], pieces[::-1])
    with pytest.raises(ValueError, match='overlaps'):
        _chk_disjoint(pieces, pieces[::-1])


def test_product_path_refuses_cpu_tensors():
    from stmi import lib, ops
    x, s = torch.zeros((1, 4, 4, 8)), torch.zeros(8)
    with pytest.raises(lib.StmiError, match='no CPU fallback'):
        ops.group_norm_fwd(x, 2, s, s)
    with pytest.raises(lib.StmiError, match='no CPU fallback'):
        ops.group_norm_bwd(x, x, 2, torch.zeros((1, 2, 2)), s, s, None, None)
    with pytest.raises(lib.StmiError, match='no CPU fallback'):
        ops.GradList([x])
