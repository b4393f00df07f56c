"""-m gpu: the fp32 form's training step from run to run."""
import copy

import pytest
import torch

from cfgs import DenseASPP121
from e2e_common import grad_report, make_batch, make_dropout_masks, make_pair

pytestmark = pytest.mark.gpu


def test_statistics_of_the_forward_pass_do_not_move_the_gradients():
    """The BatchNorm sums of the forward pass have a fixed order, so that no pre-activation next to zero changes its sign from run to run
    (each such change moves the gradient behind norm5 by 3e-4 and more at random initialisation).  What is left are the fp32 atomics of the
    backward pass, 1e-6."""
    ref, mod = make_pair(DenseASPP121.Model_CFG, randomize_bn=False)
    state = copy.deepcopy(ref.state_dict())
    x, labels = make_batch(1, 128, 256)
    masks = {k: v.cuda() for k, v in make_dropout_masks(ref, 1, torch.Generator().manual_seed(5)).items()}
    mod = mod.cuda().train().set_compute_dtype(torch.float32)
    runs, stats = [], []
    for _ in range(4):
        mod.load_state_dict(state)
        mod.train_step(x.cuda(), labels.cuda(), dropout_masks=masks)
        runs.append({n: p.grad.detach().cpu().clone() for n, p in mod.named_parameters()})
        stats.append({n: b.detach().cpu().clone() for n, b in mod.named_buffers()})
    for g, s in zip(runs[1:], stats[1:]):
        for n, b in s.items():
            assert torch.equal(b, stats[0][n]), n
        rel, cos, worst = grad_report(runs[0], g)
        assert rel < 1e-4, (rel, cos, worst)
