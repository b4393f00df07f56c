"""Class scores of logits: the log probability of given labels, the entropy, and the most probable classes, per pixel (or per row
of any classifier), with their gradient.

The reference has the arg-max (graph_seg_test.py:62,146) and the mean cross-entropy (graph_seg_main.py:216,238) of the same logits;
this is what lies between: pseudo labels with a confidence or entropy threshold, uncertainty maps, and losses of one's own --
hard-example mining, focal or weighted losses, entropy minimisation -- without full-resolution probabilities in memory.
DenseASPP.score runs it on the network's own logits.

    s = label_scores(logits, labels, top_k=3)          # logits N x C x ..., labels N x ...
    loss = -(s.logp * weight).sum() + 0.1 * s.entropy.mean()
    loss.backward()
"""
from collections import namedtuple

import torch

from . import _lib

Scores = namedtuple('Scores', 'logp entropy top_logp top_class')
Scores.__doc__ = """logp, entropy: fp32, the shape of the labels; top_logp (fp32), top_class (int64): N x top_k x ...  None if not asked for."""

MAX_TOP = _lib.SCORES_MAX_TOP


def label_scores(logits, labels=None, top_k=0, ignore_index=-100, entropy=True, upsample=1):
    """Scores(logp, entropy, top_logp, top_class) of every row of `logits`.

    logits: N x C x ... (classes in dimension 1) float32, bfloat16 or float16 on a GPU, any strides: NCHW, channels_last, or
    token x vocabulary.  All arithmetic is fp32.
    labels: int64, N x ...; logp is 0 (and sends back no gradient) where the label is ignore_index or outside [0, C).
    top_k: up to 8; the classes of the largest logits, descending, the lowest class first among equal ones.
    upsample=8: logits are N x C x h x w at 1/8 resolution, C <= 32, and the rows are the 8h x 8w pixels of their bilinear upsample
    (align_corners=False), which is never written out.

    Classes at -inf count as masked out: probability 0, never an alternative; alternatives that a row does not have are class -1
    with log probability -inf.  A row with every class masked out has logp -inf (if labelled), entropy 0 and gradient 0.  A NaN or
    +inf in a row makes its logp (if labelled), entropy and top_logp NaN and its top_class -1.  Rows whose upstream gradients
    are all 0 get gradient 0 whatever they hold.  With upsample=8, -inf meets interpolation weights of 0 as in torch's upsample (NaN):
    give finite logits there.  Its fast form takes pixels whose largest logit is below 64 in magnitude, if no class changes its distance from
    the largest by more than 33 between two low-resolution rows and all logits are below 1e5 in magnitude.  Others (a class masked by -1e9, a
    common offset of 100) cost twice as much, with the backward pass three times, along with the pixels around them.

    logp, entropy and top_logp are differentiable with respect to the logits (once, in reverse mode; dual tensors of forward mode are refused);
    the gradient has the logits' type."""
    if not isinstance(logits, torch.Tensor):
        raise TypeError('label_scores needs a tensor of logits, got %s' % type(logits).__name__)
    return Scores._make(_lib.binding().label_scores(logits, labels, top_k, ignore_index, entropy, upsample, _lib.raw_stream(logits)))
