"""-m gpu: class scores in the layouts and sizes where another kernel takes over."""
import pytest
import torch

from test_gpu_scores import _check, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('classes,pixels', [(32, 2097153), (33, 1048577), (33, 2097155)])
def test_planes_on_both_sides_of_the_class_limit(classes, pixels, dtype):
    z, labels, logits = _make((1, classes, pixels), dtype, 'dense', classes)
    _check(z, labels, logits, 1, True)
