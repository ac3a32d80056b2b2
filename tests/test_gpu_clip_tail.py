"""The ragged last batch of an epoch is clipped like the others when the trainer clips."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize('max_norm', [1.0, None], ids=['clipped', 'not clipped'])
def test_ragged_batch_is_clipped_like_the_others(cuda, max_norm):
    import full_graph_stylizer_network as F
    import numpy as np
    from oracle import tf_ops as O
    from stmi.trainer import StyleTrainer
    rng = np.random.default_rng(0)
    batch = torch.tensor(rng.random((1, 32, 24, 3)).astype(np.float32), device=cuda)
    style = torch.tensor(rng.random((1, 30, 22, 3)).astype(np.float32))
    vggw, mean = O.synthetic_vgg_weights(seed=7, width_div=8, bias_scale=0.1), np.array([103.9, 116.8, 123.7], np.float32)
    config = types.SimpleNamespace(style_weight=1e-2, content_weight=1e4, total_variation_weight=1e8)
    main = StyleTrainer(2, 32, 24, cuda, vggw, mean, 1e-2, 1e4, 1e8, params=O.init_stylizer_params(seed=1), max_grad_norm=max_norm)
    main.set_style_image(style)
    tail = F._tail_trainer({}, main, 1, vggw, mean, config, torch.float32)
    tail.step(batch)
    F._sync_back(tail, main)
    g = tail.net.flat_grad.double()
    norm = g.norm().item()
    assert norm > 2.0
    want = (1 - 0.9) * g / (norm if max_norm else 1.0)          # the first step's first moment
    assert ((main.m.double() - want).abs() <= 8 * U * want.abs() + 2.0 ** -133).all()
    if max_norm:
        assert abs(main.grad_norm.item() - norm) <= 2 * U * norm
    else:
        assert main.grad_norm is None
