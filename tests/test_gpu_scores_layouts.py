"""-m gpu: class scores in the layouts and sizes where another kernel takes over."""
import pytest
import torch

from test_gpu_scores import _check, _label_scores, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('classes,pixels', [(32, 2097153), (33, 1048577), (33, 2097155)])
def test_planes_on_both_sides_of_the_class_limit(classes, pixels, dtype):
    z, labels, logits = _make((1, classes, pixels), dtype, 'dense', classes)
    _check(z, labels, logits, 1, True)


@pytest.mark.parametrize('shape,layout', [((1, 21841), 'step_classes'), ((3, 600), 'step_classes'), ((1, 50257, 16), 'dense'), ((2, 512, 3, 5), 'dense'),
                                          ((2, 700, 9, 11), 'crop'), ((1, 512, 16384), 'dense'), ((1, 512, 16385), 'dense'), ((2, 511, 7), 'dense')])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_many_classes_that_do_not_lie_side_by_side(shape, layout, dtype):
    z, labels, logits = _make(shape, dtype, 'dense' if layout == 'step_classes' else layout, shape[1], mask='random')
    if layout == 'step_classes':                          # every second element of a row
        logits = torch.stack((logits, torch.full_like(logits, 9.0)), -1).flatten(1)[:, ::2]
        assert logits.stride(1) == 2
    _check(z, labels, logits, 5, True)
    _check(z, labels, logits, 0, True)


def test_few_rows_of_strided_classes_do_not_wait_for_one_lane():
    """A lane alone takes 2.7 and 6.5 ms for these: 30 of them in a row well below the time of three."""
    two = torch.randn(1, 2 * 21841, device='cuda')[:, ::2]
    planes = torch.randn(1, 50257, 16, device='cuda')
    for logits, limit in ((two, 8.0), (planes, 19.0)):
        for _ in range(3):
            _label_scores(logits, top_k=5)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(30):
            _label_scores(logits, top_k=5)
        b.record()
        b.synchronize()
        assert a.elapsed_time(b) < limit, a.elapsed_time(b)
