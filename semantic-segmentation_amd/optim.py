"""Fused Adam over the flat parameter arena.

Takes over torch.optim.Adam(model.parameters(), weight_decay=wd, lr=lr) with the per-epoch poly
learning-rate rule of the reference loop (graph_seg_main.py:186,241-245): one kernel updates
fp32 master weights, both moments and the bf16 shadow weights; a second rebuilds the transposed
copies the data-gradient kernels read.

Checkpoints: state_dict() / load_state_dict() speak torch.optim.Adam's format (per-parameter
``step`` / ``exp_avg`` / ``exp_avg_sq`` in model.parameters() order, one param group), so the
reference's ``'optimizer': optimizer.state_dict()`` / ``optimizer.load_state_dict(...)``
(graph_seg_main.py:199,280) round-trips between this optimizer and torch.optim.Adam.

Gradient norm and clipping: grad_norm / clip_grads_ on any list of gradient tensors, clip_grad_norm_ with the
arguments of torch.nn.utils.clip_grad_norm_, FusedAdam.step(max_grad_norm=...) and adam_update_ with the clip
coefficient applied inside the update (the gradients are read twice and not rewritten).  None of them waits
for the GPU unless error_if_nonfinite is set.
"""
import ctypes
import math
import operator

import numpy
import torch

from . import _lib


def _unwrap(model):
    return model.module if isinstance(model, torch.nn.DataParallel) else model


_DTYPE_CODE = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_MAX_PIECES = 1 << 16
_dtype_of, _requires_grad = operator.attrgetter('dtype'), operator.attrgetter('requires_grad')


def _dense_pieces(t):
    """(address, elements) of the dense pieces of a tensor whose elements do not fill one piece of memory: its dimensions are
    merged from the innermost stride outwards as far as they are contiguous, the rest is walked (expanded ones over and over)."""
    dims = sorted(((st, n) for st, n in zip(t.stride(), t.shape) if n > 1), key=lambda d: (d[0] == 0, d[0]))
    run, i = 1, 0
    while i < len(dims) and dims[i][0] == run:
        run *= dims[i][1]
        i += 1
    outer = dims[i:]
    if math.prod(n for _, n in outer) > _MAX_PIECES:
        raise ValueError('a gradient of shape %s and strides %s lies in more than %d separate pieces: make it contiguous'
                         % (tuple(t.shape), tuple(t.stride()), _MAX_PIECES))
    offs = [0]
    for st, n in reversed(outer):
        offs = [o + k * st for o in offs for k in range(n)]
    base, size = t.data_ptr(), t.element_size()
    return [(base + o * size, run) for o in offs]


class _Grads:
    """The device ranges of a list of gradient tensors and the descriptor of the norm kernels over them.  Lives for one call.

    A list of hundreds of tensors costs more host time to look at than the kernels take, so every property is read in one
    pass of C calls over the list, and the ranges travel as one array of (address, elements, type code) words, which is the layout of
    dsaspp_grad_range.  Joining neighbours and looking for overlaps is the library's."""

    def __init__(self, grads, norm_type, in_place, who):
        norm_type = float(norm_type)
        if norm_type not in (2.0, math.inf):
            raise ValueError('%s: norm_type must be 2 or inf, got %r' % (who, norm_type))
        T = torch.Tensor
        try:
            devices = set(map(T.get_device, grads))
            dtypes = set(map(_dtype_of, grads))
            dense = all(map(T.is_contiguous, grads))
            if len(devices) != 1 or -1 in devices:
                raise ValueError('%s: the gradients must be on one GPU, got %s' % (who, ', '.join(sorted({str(t.device) for t in grads}))))
            for dt in dtypes:
                if dt not in _DTYPE_CODE:
                    raise TypeError('%s needs float32, bfloat16 or float16 gradients, got %s' % (who, dt))
            if len(dtypes) == 1:
                codes = _DTYPE_CODE[next(iter(dtypes))]
            else:
                codes = [_DTYPE_CODE[t.dtype] for t in grads]
            if dense:
                ptrs, counts = list(map(T.data_ptr, grads)), list(map(T.numel, grads))
            else:
                ptrs, counts, piece_codes = [], [], []
                for t in grads:
                    if t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last)):
                        pieces = ((t.data_ptr(), t.numel()),)
                    else:
                        pieces = _dense_pieces(t) if t.numel() else ()
                    for p, n in pieces:
                        ptrs.append(p)
                        counts.append(n)
                        piece_codes.append(_DTYPE_CODE[t.dtype])
                codes = piece_codes
        except (RuntimeError, NotImplementedError) as e:
            raise TypeError('%s needs dense gradient tensors: %s' % (who, e)) from None
        self.words = words = numpy.empty((len(ptrs), 3), dtype=numpy.int64)     # read by the calls below
        if ptrs:
            words[:, 0], words[:, 1], words[:, 2] = ptrs, counts, codes
        if 0 in counts:
            self.words = words = numpy.ascontiguousarray(words[words[:, 1] != 0])
        dev = devices.pop()
        d = self.desc = _lib.clip_desc(words.ctypes.data, len(words), 2 if norm_type == 2.0 else 0, 1.0, 0.0)
        self.lib = lib = _lib.load()
        if in_place and lib.dsaspp_grad_ranges_overlap(ctypes.byref(d)) != 0:
            raise ValueError('%s: two gradients (or two elements of one) share memory: each would be scaled twice' % who)
        need = lib.dsaspp_grad_norm_workspace(ctypes.byref(d))
        if need < 0:
            raise _lib.DsasppError(lib.dsaspp_last_error().decode())
        # from the caching allocator for this call: two calls, streams or captured graphs never share a workspace
        device = grads[0].device
        self.ws = torch.empty(need, dtype=torch.float64, device=device)
        self.norm = torch.empty((), dtype=torch.float32, device=device)
        d.ws, d.ws_len, d.norm = self.ws.data_ptr(), need, self.norm.data_ptr()
        self.stream = _lib.raw_stream(dev)

    def call(self, name):
        _lib.check(getattr(self.lib, name)(ctypes.byref(self.desc), self.stream))


def _written(tensors):
    """Tell autograd that the kernels wrote these tensors, as torch's own in-place operations do."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:                       # tensors made in inference mode have no version
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _checked(grads, who):
    """The gradients as a list of GPU tensors."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    for kind in set(map(type, grads)):
        if not issubclass(kind, torch.Tensor):
            raise TypeError('%s needs tensors, got %s' % (who, kind.__name__))
    if grads and not grads[0].is_cuda:
        raise ValueError('%s needs gradients on a GPU, got %s' % (who, grads[0].device))
    return grads


def grad_norm(grads, norm_type=2.0):
    """Global norm of a list of gradient tensors (or of one): sqrt of the sum of all squares, or the largest magnitude for
    norm_type=inf, as a 0-dim fp32 tensor on their GPU.  float32, bfloat16 and float16 tensors may be mixed.  The sums are fp64:
    magnitudes whose squares leave the fp32 range count in full, and the same tensors give the same bits each time."""
    grads = _checked(grads, 'grad_norm')
    if not grads:
        return torch.tensor(0.0)
    with _lib.on_device(grads[0]):
        g = _Grads(grads, norm_type, False, 'grad_norm')
        g.call('dsaspp_grad_norm_partials')
        g.call('dsaspp_grad_norm_finish')
    return g.norm


def clip_grads_(grads, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale every tensor of `grads` in place by min(1, max_norm / (norm + 1e-6)) with norm = grad_norm(grads, norm_type), and
    return the norm (0-dim fp32 tensor on the GPU).  A NaN norm makes every gradient NaN, as torch's clipping does, unless
    error_if_nonfinite is set: then the call waits for the norm and raises RuntimeError before it writes anything.
    Tensors that share memory are refused."""
    grads = _checked(grads, 'clip_grads_')
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError('clip_grads_: max_norm must be >= 0, got %r' % max_norm)
    if not grads:
        return torch.tensor(0.0)
    if any(map(_requires_grad, grads)):
        raise ValueError('clip_grads_ writes plain gradient tensors in place; a tensor that requires grad is not one (pass p.grad, or '
                         'use clip_grad_norm_ on the parameters)')
    with _lib.on_device(grads[0]):
        g = _Grads(grads, norm_type, True, 'clip_grads_')
        g.desc.max_norm = max_norm
        if error_if_nonfinite:
            g.call('dsaspp_grad_norm_partials')
            g.call('dsaspp_grad_norm_finish')
            if not math.isfinite(float(g.norm)):
                raise RuntimeError('the norm of the gradients is not finite (%r): nothing was clipped' % float(g.norm))
            g.call('dsaspp_clip_scale')
        else:
            g.call('dsaspp_clip_grads')
    _written(grads)
    return g.norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ on these kernels: clip_grads_ over the .grad of the parameters that have one.  `foreach` is
    accepted and has no effect.  After a GradReducer the arena holds summed gradients until FusedAdam.step divides
    them: clip with step(max_grad_norm=...) there, or call average_grads() first."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite)


def adam_update_(param, grad, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, grad_scale=1.0,
                 max_grad_norm=math.inf, norm_type=2.0, shadow=None):
    """One Adam update of a flat parameter, in place, on grad * grad_scale * coef with the clip coefficient
    coef = min(1, max_grad_norm / (norm + 1e-6)), norm = grad_scale * grad_norm(grad).  Returns the norm (0-dim fp32 tensor).
    param, grad, exp_avg, exp_avg_sq: contiguous float32 tensors of one size on one GPU; `step` counts from 1;
    `shadow`: a bfloat16 tensor that receives the rounded parameters."""
    tensors = [param, grad, exp_avg, exp_avg_sq]
    for t in tensors:
        if t.dtype != torch.float32 or t.numel() != param.numel() or t.device != param.device or not t.is_contiguous() or not t.is_cuda:
            raise ValueError('adam_update_ needs contiguous float32 tensors of one size on one GPU')
    if shadow is not None:
        if (shadow.dtype != torch.bfloat16 or shadow.numel() != param.numel() or shadow.device != param.device
                or not shadow.is_contiguous()):
            raise ValueError('adam_update_: shadow must be a contiguous bfloat16 tensor of the size of param')
        tensors.append(shadow)
    if param.numel() == 0:
        raise ValueError('adam_update_ needs at least one element')
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError('adam_update_: two of the tensors share memory')
    if int(step) < 1:
        raise ValueError('adam_update_: step counts from 1, got %r' % (step,))
    if not (0.0 < float(grad_scale) < math.inf):
        raise ValueError('adam_update_: grad_scale must be positive and finite, got %r' % (grad_scale,))
    if not float(max_grad_norm) >= 0.0:
        raise ValueError('adam_update_: max_grad_norm must be >= 0, got %r' % (max_grad_norm,))
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError('adam_update_: betas must be in [0, 1), got %r' % (betas,))
    with _lib.on_device(param):
        c = _Grads([grad], norm_type, False, 'adam_update_')
        c.desc.scale, c.desc.max_norm = float(grad_scale), float(max_grad_norm)
        c.call('dsaspp_grad_norm_partials')
        d = _lib.adam_clip_desc()
        d.n = param.numel()
        d.p, d.g, d.m, d.v = param.data_ptr(), grad.data_ptr(), exp_avg.data_ptr(), exp_avg_sq.data_ptr()
        d.w16 = None if shadow is None else shadow.data_ptr()
        d.lr, d.beta1, d.beta2, d.eps, d.weight_decay = float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay)
        d.step = int(step)
        _lib.check(c.lib.dsaspp_adam_step_clipped(ctypes.byref(d), ctypes.byref(c.desc), c.stream))
    _written([t for t in tensors if t is not grad])
    return c.norm


class FusedAdam:
    def __init__(self, model, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        self.model = _unwrap(model)
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.step_count = 0
        self.m = None
        self.v = None
        # the reference loop rewrites param_group['lr'] every step; the other entries mirror torch.optim.Adam's group
        self.param_groups = [dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, amsgrad=False,
                                  maximize=False, foreach=None, capturable=False, differentiable=False, fused=None)]

    @staticmethod
    def poly_lr(base_lr, epoch, num_epochs, power=0.9):
        return base_lr * ((1 - epoch / num_epochs) ** power)

    @property
    def global_step(self):
        """Optimizer steps taken so far (what the reference stores as checkpoint['global_step'])."""
        return self.step_count

    def zero_grad(self, set_to_none=False):
        self.model._gflat_zero()

    def _moments(self):
        flat = self.model._flat
        if self.m is None or self.m.data_ptr() == 0 or self.m.device != flat.device or self.m.numel() != flat.numel():
            m, v = torch.zeros_like(flat), torch.zeros_like(flat)
            if self.m is not None and self.m.numel() == flat.numel():     # the model moved: the moments follow it
                m.copy_(self.m)
                v.copy_(self.v)
            self.m, self.v = m, v

    def step(self, grad_scale=None, max_grad_norm=None):
        """One Adam update from the flat gradient arena.  grad_scale multiplies the gradients first; by default it is
        what the last GradReducer.run_backward left on the model (1 / world size after a summing all-reduce), else 1.
        With max_grad_norm the scaled gradients are clipped to that global Euclidean norm inside the update (the arena keeps
        what it held) and the norm before clipping is returned as a 0-dim tensor on the GPU."""
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError('FusedAdam.step: max_grad_norm must be >= 0, got %r' % (max_grad_norm,))
        if max_grad_norm is not None and grad_scale is not None and not 0.0 < float(grad_scale) < math.inf:
            raise ValueError('FusedAdam.step: with max_grad_norm the gradient scale must be positive and finite, got %r' % (grad_scale,))
        mod = self.model
        mod._check_arena()
        flat = mod._flat
        self._moments()
        if grad_scale is None:
            grad_scale = getattr(mod, '_grad_scale', 1.0)
        # the scale a GradReducer left belongs to the gradients of THAT backward pass: used once, then back to 1, so
        # that a later step on locally computed gradients (train_step without a reducer, loss.backward()) is not scaled
        mod._grad_scale = 1.0
        g0 = mod._first_param.grad
        if g0 is None or g0.data_ptr() != mod._gflat.data_ptr() + 4 * mod.arena.by_name[mod._param_names[0]].off:
            mod.sync_grads_to_arena()         # gradients came from loss.backward() through model(x), not from train_step
        self.step_count += 1
        lib = _lib.load()
        g = self.param_groups[0]
        # fp32 compute mode: the "shadow" IS the master arena (the fp32 kernels read it directly); writing packed bf16
        # there would overwrite the parameters
        shadow_is_master = mod._w16 is None or mod._w16.data_ptr() == flat.data_ptr() or mod._w16.dtype != torch.bfloat16
        if max_grad_norm is not None:
            with torch.cuda.device(flat.device):
                norm = adam_update_(flat, mod._gflat, self.m, self.v, self.step_count, lr=float(g['lr']), betas=g.get('betas', self.betas),
                                    eps=float(g.get('eps', self.eps)), weight_decay=float(g.get('weight_decay', self.weight_decay)),
                                    grad_scale=float(grad_scale), max_grad_norm=float(max_grad_norm),
                                    shadow=None if shadow_is_master else mod._w16)
                mod._get_backend().refresh_weights(mod, cast=shadow_is_master)
            mod._weights_fresh = True
            return norm
        d = _lib.adam_desc()
        d.n = flat.numel()
        d.p, d.g, d.m, d.v = flat.data_ptr(), mod._gflat.data_ptr(), self.m.data_ptr(), self.v.data_ptr()
        d.w16 = None if shadow_is_master else mod._w16.data_ptr()
        d.lr = float(g['lr'])
        d.beta1, d.beta2 = g.get('betas', self.betas)
        d.eps, d.weight_decay = float(g.get('eps', self.eps)), float(g.get('weight_decay', self.weight_decay))
        d.step = self.step_count
        d.grad_scale = float(grad_scale)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _lib.check(lib.dsaspp_adam_step(ctypes.byref(d), stream))
        mod._get_backend().refresh_weights(mod, cast=shadow_is_master)
        mod._weights_fresh = True

    # ------------------------------------------------------------------ checkpoint format of torch.optim.Adam
    def state_dict(self):
        mod = self.model
        names = mod._param_names
        state = {}
        if self.m is not None and self.step_count > 0:
            for i, n in enumerate(names):
                state[i] = dict(step=torch.tensor(float(self.step_count)),
                                exp_avg=mod.arena.view(self.m, n).clone(),
                                exp_avg_sq=mod.arena.view(self.v, n).clone())
        group = dict(self.param_groups[0])
        group['params'] = list(range(len(names)))
        return dict(state=state, param_groups=[group])

    def load_state_dict(self, sd):
        mod = self.model
        names = mod._param_names
        groups = sd['param_groups']
        ids = [i for g in groups for i in g['params']]
        if len(ids) != len(names):
            raise ValueError('optimizer state holds %d parameters, the model has %d' % (len(ids), len(names)))
        g0 = {k: v for k, v in groups[0].items() if k != 'params'}
        for g in groups[1:]:
            for k in ('lr', 'betas', 'eps', 'weight_decay'):
                if k in g and g[k] != g0.get(k):
                    raise ValueError('FusedAdam keeps one parameter group; the loaded groups differ in %r' % k)
        self.param_groups[0].update(g0)
        self.betas = tuple(self.param_groups[0]['betas'])
        self.eps, self.weight_decay = self.param_groups[0]['eps'], self.param_groups[0]['weight_decay']
        state = sd.get('state', {})
        mod._check_arena()
        self.m = None
        self._moments()
        self.step_count = 0
        if state:
            steps = set()
            named = dict(mod.named_parameters())
            for pos, pid in enumerate(ids):
                st = state.get(pid)
                if st is None:
                    raise ValueError('optimizer state has no entry for parameter %d (%s)' % (pid, names[pos]))
                if tuple(st['exp_avg'].shape) != tuple(named[names[pos]].shape):
                    raise ValueError('optimizer state of %s has shape %s, the parameter %s'
                                     % (names[pos], tuple(st['exp_avg'].shape), tuple(named[names[pos]].shape)))
                mod.arena.view(self.m, names[pos]).copy_(st['exp_avg'])
                mod.arena.view(self.v, names[pos]).copy_(st['exp_avg_sq'])
                steps.add(int(float(st['step'])))
            if len(steps) != 1:
                raise ValueError('FusedAdam keeps one step counter; the loaded state has steps %s' % sorted(steps))
            self.step_count = steps.pop()
