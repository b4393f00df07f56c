"""-m gpu: calls of the class-score and gradient-norm operators beside the usual ones."""
import pytest

from test_gpu_scores import _tiny

pytestmark = pytest.mark.gpu


def test_network_backward_after_scores_of_the_same_batch_is_refused():
    """Logits and scores of one batch share the engine's buffers: the earlier one's backward pass is refused, alone and in a common loss."""
    from e2e_common import make_batch
    _, mod = _tiny(True)
    x, labels = make_batch(1, 64, 64)
    for both in (False, True):
        out = mod(x.cuda())
        s = mod.score(x.cuda(), labels.cuda())
        loss = out.square().mean()
        with pytest.raises(RuntimeError, match='another pass'):
            (loss + s.entropy.mean() if both else loss).backward()
    s = mod.score(x.cuda(), labels.cuda())
    mod(x.cuda())
    with pytest.raises(RuntimeError, match='another pass'):
        s.entropy.mean().backward()
