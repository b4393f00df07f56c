"""-m gpu: accuracy of the x8-upsampled class scores where rounding shows.  The definition in 64 bits is that of tests/scores_ref.py, on the
interpolated logits whose every product and sum is rounded to fp32."""
import pytest
import torch

import scores_ref as R
from test_gpu_scores import _check8, _label_scores, _make8, _place

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


@pytest.mark.parametrize('offset', [64.0, -70.0, 1.0e3, -1.0e3, 1.0e4, -1.0e4, 9.0e4])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_common_offset_costs_no_accuracy(offset, dtype, monkeypatch):
    """All logits raised alike: the errors are those of an fp32 log-softmax of the interpolated logits, without a part that grows with
    their magnitude."""
    import test_gpu_scores
    monkeypatch.setattr(test_gpu_scores, '_size', lambda low: 0.0)
    z, labels, _ = _make8((2, 19, 5, 20), torch.float32, 'last', 3)
    z = ((z * 0.75).clamp(-5.5, 5.5) + offset).to(dtype)
    _check8(z, labels, _place(z, 'last'), 3, True)
    _check8(z, labels, _place(z, 'dense'), 0, True)


@pytest.mark.parametrize('x', [2, 7, 8, 12, 15, 16])
@pytest.mark.parametrize('offset', [100.0, -100.0])
def test_pixels_with_an_offset_beside_ordinary_ones(x, offset):
    """The two passes, whose waves hold different columns, do not agree about which form a column takes."""
    z, labels, _ = _make8((1, 19, 6, 20), torch.float32, 'last', 7)
    z[:, :, :, x] += offset
    for layout in ('last', 'dense'):
        _check8(z, labels, _place(z, layout), 2, True)
        _check8(z, labels, _place(z, layout), 0, True)


@pytest.mark.parametrize('mask', [-100.0, -3.0e4, -1.0e9])
def test_finite_masks_of_whole_classes(mask, monkeypatch):
    """Classes masked by a large negative number in every pixel.  100 below the others p is 2^-144: a term of the gradient has a spacing of
    2^-149 there in place of a relative rounding, and a low-resolution pixel adds up to 256 terms with four roundings each."""
    monkeypatch.setattr(R, 'tiny', lambda dtype: 1024 * 2.0 ** -149)
    z, labels, _ = _make8((1, 19, 6, 20), torch.float32, 'last', 5)
    z[:, 4:9] = mask
    _check8(z, labels, _place(z, 'last'), 3, True)
    _check8(z, labels, _place(z, 'dense'), 0, True)
