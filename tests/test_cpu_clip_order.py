"""The clipped update needs the norm of its gradients first.  No GPU: a list without one is refused before anything is launched."""
import pytest
import torch


def test_update_without_a_norm_is_refused():
    from stmi import ops
    lst = ops.GradList.__new__(ops.GradList)
    lst._summed = False
    t = torch.zeros(4)
    with pytest.raises(ValueError, match='sum_squares'):
        ops.adam_tf1(t, t, t, t, 1e-3, t=1, clip=lst, max_norm=1.0)
