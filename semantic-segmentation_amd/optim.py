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

import torch

from . import _lib


def _unwrap(model):
    return model.module if isinstance(model, torch.nn.DataParallel) else model


def _list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _stream(tensors):
    """Current stream of the first tensor's GPU; anything that is no tensor is left to the binding's checks."""
    t = tensors[0] if tensors else None
    return _lib.raw_stream(t) if isinstance(t, torch.Tensor) else 0


def grad_norm(grads, norm_type=2.0):
    """Global norm of a list of gradient tensors (or of one): sqrt of the sum of all squares, or the largest magnitude for
    norm_type=inf, as a 0-dim fp32 tensor on their GPU.  float32, bfloat16 and float16 tensors may be mixed.  The sums are fp64:
    magnitudes whose squares leave the fp32 range count in full, and the same tensors give the same bits each time.  The result carries
    no gradient of its own."""
    grads = _list(grads)
    return _lib.binding().grad_norm(grads, norm_type, _stream(grads))


def clip_grads_(grads, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale every tensor of `grads` in place by min(1, max_norm / (norm + 1e-6)) with norm = grad_norm(grads, norm_type), and
    return the norm (0-dim fp32 tensor on the GPU).  A NaN norm makes every gradient NaN, as torch's clipping does, unless
    error_if_nonfinite is set: then the call waits for the norm and raises RuntimeError before it writes anything.
    Tensors that share memory are refused."""
    grads = _list(grads)
    return _lib.binding().clip_grads(grads, False, max_norm, norm_type, error_if_nonfinite, _stream(grads))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ on these kernels: clip_grads_ over the .grad of the parameters that have one.  `foreach` is
    accepted and has no effect.  After a GradReducer the arena holds summed gradients until FusedAdam.step divides
    them: clip with step(max_grad_norm=...) there, or call average_grads() first."""
    parameters = _list(parameters)
    first = next((p for p in parameters if getattr(p, 'grad', None) is not None), None)
    return _lib.binding().clip_grads(parameters, True, max_norm, norm_type, error_if_nonfinite, 0 if first is None else _lib.raw_stream(first.grad))


def adam_update_(param, grad, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, grad_scale=1.0,
                 max_grad_norm=math.inf, norm_type=2.0, shadow=None):
    """One Adam update of a flat parameter, in place, on grad * grad_scale * coef with the clip coefficient
    coef = min(1, max_grad_norm / (norm + 1e-6)), norm = grad_scale * grad_norm(grad).  Returns the norm (0-dim fp32 tensor).
    param, grad, exp_avg, exp_avg_sq: contiguous float32 tensors of one size on one GPU; `step` counts from 1;
    `shadow`: a bfloat16 tensor that receives the rounded parameters."""
    return _lib.binding().adam_update(param, grad, exp_avg, exp_avg_sq, step, lr, betas[0], betas[1], eps, weight_decay, grad_scale,
                                      max_grad_norm, norm_type, shadow, _lib.raw_stream(param))


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
        g0 = mod._first_param.grad
        if g0 is None or g0.data_ptr() != mod._gflat.data_ptr() + 4 * mod.arena.by_name[mod._param_names[0]].off:
            mod.sync_grads_to_arena()         # gradients came from loss.backward() through model(x), not from train_step
        step = self.step_count + 1            # counted once the update has been launched: a refused one changes nothing
        lib = _lib.load()
        g = self.param_groups[0]
        # fp32 compute mode: the "shadow" IS the master arena (the fp32 kernels read it directly); writing packed bf16
        # there would overwrite the parameters
        shadow_is_master = mod._w16 is None or mod._w16.data_ptr() == flat.data_ptr() or mod._w16.dtype != torch.bfloat16
        if max_grad_norm is not None:
            with torch.cuda.device(flat.device):
                norm = adam_update_(flat, mod._gflat, self.m, self.v, step, lr=float(g['lr']), betas=g.get('betas', self.betas),
                                    eps=float(g.get('eps', self.eps)), weight_decay=float(g.get('weight_decay', self.weight_decay)),
                                    grad_scale=float(grad_scale), max_grad_norm=float(max_grad_norm),
                                    shadow=None if shadow_is_master else mod._w16)
                self._counted(step)
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
        d.step = step
        d.grad_scale = float(grad_scale)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _lib.check(lib.dsaspp_adam_step(ctypes.byref(d), stream))
        self._counted(step)
        mod._get_backend().refresh_weights(mod, cast=shadow_is_master)
        mod._weights_fresh = True

    def _counted(self, step):
        self.step_count = step
        # the scale a GradReducer left belongs to the gradients of THAT backward pass: used once, then back to 1, so
        # that a later step on locally computed gradients (train_step without a reducer, loss.backward()) is not scaled
        self.model._grad_scale = 1.0

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
