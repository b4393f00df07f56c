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


@pytest.mark.parametrize('hi,lo,rest', [(22.1, -22.9, -35.0), (10.0, -12.0, -14.0), (60.0, -60.0, -61.0), (3.0, -0.5, -4.0)])
def test_two_classes_that_all_but_tie_far_below_the_leading_one(hi, lo, rest):
    """Classes 0 and 30 a few steps of the last place apart, class 31 far above them: the order is that of the logits to the bit."""
    for seed in range(2):
        g = torch.Generator().manual_seed(seed)
        n = (1, 64, 65)
        z = rest + torch.randn(1, 32, 64, 65, generator=g) * 0.1
        base = lo + torch.randn(n, generator=g) * 0.3
        z[:, 31] = hi + torch.randn(n, generator=g) * 0.3
        z[:, 0] = base + torch.randn(n, generator=g) * abs(lo) * 2.0e-7
        z[:, 30] = base + torch.randn(n, generator=g) * abs(lo) * 2.0e-7
        s = _label_scores(_place(z, 'last'), top_k=3, upsample=8)
        full = R.interpolate(z)
        want = torch.sort(full, dim=1, descending=True, stable=True).indices[:, :3]
        assert torch.equal(s.top_class.cpu(), want), int((s.top_class.cpu() != want).any(1).sum())
        assert bool((s.top_logp[:, 1:] <= s.top_logp[:, :-1]).all())
