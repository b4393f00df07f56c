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
import ctypes
from collections import namedtuple

import torch

from . import _lib

Scores = namedtuple('Scores', 'logp entropy top_logp top_class')
Scores.__doc__ = """logp, entropy: fp32, the shape of the labels; top_logp (fp32), top_class (int64): N x top_k x ...  None if not asked for."""

_DTYPE_CODE = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
MAX_TOP = _lib.SCORES_MAX_TOP
MAX_CLASSES_UPSAMPLED = 32


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _call(name, d, t):
    lib = _lib.load()
    with torch.cuda.device(t.device):
        _lib.check(getattr(lib, name)(ctypes.byref(d), _stream(t)))


def _row_strides(shape, strides):
    """Row dimensions (without the classes) merged into at most three (size, stride) pairs, the first of them dimension 0 by
    itself; None if they do not merge that far."""
    rest = []
    for n, st in zip(shape[2:], strides[2:]):
        if n == 1:
            continue
        if rest and rest[-1][1] == n * st:
            rest[-1] = (rest[-1][0] * n, st)
        else:
            rest.append((n, st))
    if len(rest) > 2:
        return None
    rest = [(1, 0)] * (2 - len(rest)) + rest
    return [(shape[0], strides[0])] + rest


def _upstream(d, name, g):
    """An upstream gradient for the kernels: dense, or one value for all (what .sum() and .mean() send back)."""
    if g is None:
        return None
    g = g.float()
    one = all(st == 0 or n == 1 for n, st in zip(g.shape, g.stride()))
    if not one:
        g = g.contiguous()
    setattr(d, name, g.data_ptr())
    setattr(d, name + '_one', int(one))
    return g


class _Plan:
    """Checked arguments of one call on logits of this shape and device, and its passes."""

    def __init__(self, shape, device, labels, top_k, ignore_index, entropy, upsample):
        shape = tuple(shape)
        if device.type != 'cuda':
            raise ValueError('label_scores needs logits on a GPU')
        if upsample not in (1, 8):
            raise ValueError('upsample must be 1 or 8, got %r' % (upsample,))
        if len(shape) < 2 or (upsample == 8 and len(shape) != 4):
            raise ValueError('logits must be N x C x ...%s, got %s' % (' (N x C x h x w with upsample=8)' if upsample == 8 else '', shape))
        n, c = shape[:2]
        top_k = int(top_k)
        if c < 1 or c >= 1 << 30 or (upsample == 8 and c > MAX_CLASSES_UPSAMPLED):
            raise ValueError('%d classes: at least one%s' % (c, ', at most %d with upsample=8' % MAX_CLASSES_UPSAMPLED if upsample == 8 else ''))
        if not 0 <= top_k <= min(MAX_TOP, c):
            raise ValueError('top_k must be in [0, %d] and at most the %d classes, got %d' % (MAX_TOP, c, top_k))
        if labels is None and not entropy and top_k == 0:
            raise ValueError('nothing to compute: no labels, no entropy, top_k = 0')
        rows = shape[2:]
        if upsample == 8:
            rows = tuple(8 * v for v in rows)
        self.rows, self.tail = (n,) + rows, rows
        if labels is not None:
            if labels.dtype != torch.int64 or tuple(labels.shape) != self.rows or labels.device != device:
                raise ValueError('labels must be an int64 tensor of shape %s on the device of the logits' % (self.rows,))
            labels = labels.contiguous()
        self.n, self.c, self.top_k, self.labels, self.entropy, self.upsample = n, c, top_k, labels, bool(entropy), upsample
        self.ignore_index = int(ignore_index)
        self.empty = 0 in shape

    def desc(self, logits):
        """Descriptor over `logits` (strided as they are) and the tensor that it points to."""
        if self.upsample == 8:
            d = _lib.scores8_desc()
            d.n_img, d.h, d.w = self.n, logits.shape[2], logits.shape[3]
            d.sn, d.sc, d.sy, d.sx = logits.stride()
        else:
            dims = _row_strides(logits.shape, logits.stride())
            if dims is None:                          # rows scattered over more than three strides
                logits = logits.contiguous()
                dims = _row_strides(logits.shape, logits.stride())
            d = _lib.scores_desc()
            (d.d0, d.s0), (d.d1, d.s1), (d.d2, d.s2) = dims
            d.sc = logits.stride(1)
        d.dtype, d.n_class, d.top_k = _DTYPE_CODE[logits.dtype], self.c, self.top_k
        d.logits, d.labels, d.ignore_index = logits.data_ptr(), _ptr(self.labels), self.ignore_index
        return d, logits

    def forward(self, logits, need_stats):
        d, logits = self.desc(logits)
        new = dict(device=logits.device)
        logp = torch.empty(self.rows, dtype=torch.float32, **new) if self.labels is not None else None
        ent = torch.empty(self.rows, dtype=torch.float32, **new) if self.entropy else None
        top_logp = top_class = stats = None
        if self.top_k:
            shape = (self.n, self.top_k) + self.tail
            top_logp = torch.empty(shape, dtype=torch.float32, **new)
            top_class = torch.empty(shape, dtype=torch.int64, **new)
        if need_stats and self.upsample == 1:
            stats = torch.empty(self.rows + (2,), dtype=torch.float32, **new)
            d.stats = stats.data_ptr()
        d.logp, d.entropy, d.top_logp, d.top_class = _ptr(logp), _ptr(ent), _ptr(top_logp), _ptr(top_class)
        if not self.empty:
            _call('dsaspp_scores8_fwd' if self.upsample == 8 else 'dsaspp_scores_fwd', d, logits)
        return Scores(logp, ent, top_logp, top_class), stats

    def backward(self, logits, stats, entropy, top_class, g_logp, g_entropy, g_top, out=None):
        """Gradient of the logits in their shape and type; `out`: a tensor of that shape, any strides, that receives it
        (upsample=8 only)."""
        d, logits = self.desc(logits)
        up = [_upstream(d, 'g_logp', g_logp), _upstream(d, 'g_entropy', g_entropy), _upstream(d, 'g_top', g_top)]
        d.entropy, d.top_class = _ptr(entropy), _ptr(top_class)
        shape, ws = logits.shape, None
        if self.upsample == 8:
            if out is None:
                out = _like(logits)
            d.dlogits, d.g_dtype = out.data_ptr(), _DTYPE_CODE[out.dtype]
            d.gn, d.gc, d.gy, d.gx = out.stride()
            ws = torch.empty(max(_lib.load().dsaspp_scores8_workspace(ctypes.byref(d)), 0), dtype=torch.float32, device=logits.device)
            d.ws, d.ws_len = ws.data_ptr(), ws.numel()
            name = 'dsaspp_scores8_bwd'
        else:
            d.stats = _ptr(stats)
            # dense in the order of the kernel that runs: classes innermost if the logits have them so, else the logits' own shape
            if d.sc == 1 or self.c == 1:
                out = torch.empty(self.rows + (self.c,), dtype=logits.dtype, device=logits.device).movedim(-1, 1)
            else:
                out = torch.empty(shape, dtype=logits.dtype, device=logits.device)
            d.dlogits = out.data_ptr()
            name = 'dsaspp_scores_bwd'
        if not self.empty:
            if all(u is None for u in up):
                out.zero_()
            else:
                _call(name, d, logits)
        del up, ws                                     # in use until here; freed in the order of the stream
        return out


def _like(logits):
    """An empty tensor of the shape and type of the logits, classes innermost if theirs are."""
    if logits.stride(1) == 1 and logits.shape[1] > 1:
        return torch.empty((logits.shape[0],) + tuple(logits.shape[2:]) + (logits.shape[1],), dtype=logits.dtype, device=logits.device).movedim(-1, 1)
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


class _LabelScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, plan):
        s, stats = plan.forward(logits, True)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        # the labels too: autograd then notices if any of them is overwritten before the backward pass
        ctx.save_for_backward(logits, stats, s.entropy, s.top_class, plan.labels)
        if s.top_class is not None:
            ctx.mark_non_differentiable(s.top_class)
        return tuple(s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        logits, stats, entropy, top_class, _ = ctx.saved_tensors
        return ctx.plan.backward(logits, stats, entropy, top_class, g_logp, g_entropy, g_top), None


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
    give finite logits there.

    logp, entropy and top_logp are differentiable with respect to the logits (once); the gradient has the logits' type."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPE_CODE:
        raise TypeError('logits must be a float32, bfloat16 or float16 tensor, got %s' % (logits.dtype if isinstance(logits, torch.Tensor) else type(logits).__name__))
    plan = _Plan(logits.shape, logits.device, labels, top_k, ignore_index, entropy, upsample)
    if torch.is_grad_enabled() and logits.requires_grad:
        return Scores(*_LabelScores.apply(logits, plan))
    return plan.forward(logits, False)[0]
