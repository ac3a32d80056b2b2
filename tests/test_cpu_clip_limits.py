"""How long a gradient list may be.  A block's index of a chunk is an int that runs past the last chunk by up to a grid's
2048 blocks: lists that would carry it past 2^31 are refused.  No GPU."""
import ctypes


def test_lists_whose_index_would_overflow_are_refused():
    from stmi import lib
    h = lib.load()
    most = 2 ** 31 - 4096
    assert most + lib.GRAD_WS_DOUBLES < 2 ** 31
    for chunks in (most + 1, 2 ** 31 - 2048, 2 ** 31 - 1, 2 ** 31 + 5):
        counts, dtypes = (ctypes.c_long * 1)(chunks * 4096), (ctypes.c_int * 1)(lib.F32)
        assert h.stmi_grad_list_chunks(counts, dtypes, 1) == chunks
        place = (ctypes.c_void_p * 1)(1 << 40)
        # refused before the table is touched
        assert h.stmi_grad_list_fill(place, place, counts, dtypes, 1, ctypes.byref(lib.GradChunk())) == -1
        assert b'chunks' in h.stmi_last_error()
    for n in (most + 1, 2 ** 31 - 1):
        assert h.stmi_grad_sum_squares(1, n, 1, None) == -1
        assert h.stmi_grad_norm(1, n, 1, 1, None) == -1
        assert h.stmi_grad_clip(1, n, 1, 1.0, 1, None) == -1
        assert h.stmi_adam_tf1_clip(1, 1, 1, 1, 8, 1e-3, .9, .999, 1e-8, 1.0, 1, n, 1.0, None, None, 1, None) == -1


def test_outputs_beside_the_tensors_are_taken():
    import torch
    from stmi.ops import _chk_disjoint
    a, b = torch.zeros(100), torch.zeros(100)
    _chk_disjoint([a], [b])
    _chk_disjoint([a[:50], b[50:]], [a[50:], b[:50]])
