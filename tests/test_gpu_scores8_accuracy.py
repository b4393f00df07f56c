"""-m gpu: accuracy of the x8-upsampled class scores where rounding shows.  The definition in 64 bits is that of tests/scores_ref.py, on the
interpolated logits whose every product and sum is rounded to fp32."""
import pytest
import torch

import scores_ref as R
from test_gpu_scores import _label_scores, _place

pytestmark = pytest.mark.gpu
U = R.U


@pytest.mark.parametrize('classes', [5, 19, 30])
@pytest.mark.parametrize('lead', [15.0, 20.0, 30.0, 57.0, 100.0, 200.0])
@pytest.mark.parametrize('train', [False, True])
def test_confident_pixels_have_log_probabilities_of_at_most_zero(classes, lead, train):
    """One class leads every pixel by at least lead - 12, the others lie within 6 of 0.  The leading class then is the reference of every
    exponential and its own term is 1, so that log p = -log s: s takes one rounding of at most 2 U per class (log p of 30 others 3 below is
    above -1), the logarithm and the products with it at most 8 U together.  What the rounding of a logit (15 R half-steps at most, of both)
    and the products down a cell (23) do to the other classes counts by their share 1 - p."""
    g = torch.Generator().manual_seed(classes)
    z = (torch.randn(2, classes, 9, 21, generator=g) * 3).clamp(-6, 6)
    z[:, 0] += lead
    labels = torch.zeros(2, 72, 168, dtype=torch.int64)
    low = _place(z, 'last').requires_grad_(train)
    s = _label_scores(low, labels.cuda(), top_k=2, upsample=8)
    assert bool((s.logp <= 0).all()) and bool((s.top_logp <= 0).all()) and bool((s.entropy >= 0).all())
    assert bool(torch.isfinite((1 - s.logp.exp()) ** 1.5).all())
    r = R.scores(R.interpolate(z), labels, 2, -100, classes)
    rest = -torch.expm1(r['logp'])
    lim = (2 * classes + 8) * U + rest * U * (2 * 15 * (lead + 6) + 23)
    R.agree(s.logp, r['logp'], lim, 'logp')
    assert torch.equal(s.top_class.cpu(), r['top_class'])
    R.agree(s.top_logp[:, 0], r['top_logp'][:, 0], lim, 'top_logp')
