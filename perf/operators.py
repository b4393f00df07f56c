"""Cases of the class-score operators (log probabilities of given labels, entropy, top alternatives, their gradient) and of
the gradient-norm operators (clipping by the global norm, the clipped Adam update), each in a plain torch form and as the calls
that a program makes of this package.

    own = False    run() computes the plain form: elementary torch operations in 32 bits
    own = True     run() calls semantic_segmentation_amd

A case is a dict.  op "scores": logits [shape], class axis at dim 1 after `last` (True: the classes are the contiguous axis,
the tensor is handed over as a view with its class axis moved to dim 1).  op "scores8": low-resolution logits that the
operator interpolates by 8.  op "clip" / "adam": gradients of many tensors in one buffer, every tensor starting at
a multiple of 8 elements.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
IGNORE = -100
EPS = 1e-6          # what clipping adds to the norm, as torch.nn.utils.clip_grad_norm_ does


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one pixel (a click, a single token) against a large open vocabulary of classes: latency
        dict(name='scores_one_row', op='scores', rows=1, classes=21841, inner=1, last=True, dtype='bf16', top_k=5, train=False, masked=0.0),
        # a head that leaves NHWC scores: 150 classes, odd crop of 473 x 473
        dict(name='scores_rows_150', op='scores', rows=473 * 473, classes=150, inner=1, last=True, dtype='bf16', top_k=3, train=False, masked=0.1),
        # training on region features against 1203 classes, some of them masked out, odd row count
        dict(name='scores_rows_1203_train', op='scores', rows=8191, classes=1203, inner=1, last=True, dtype='fp32', top_k=0, train=True, masked=0.2),
        # the logits that model(x) returns: 19 classes NCHW fp32, two 1024 x 2048 images, labels with their alternatives
        dict(name='scores_planes_19', op='scores', rows=2, classes=19, inner=1024 * 2048, last=False, dtype='fp32', top_k=3, train=False, masked=0.0),
        # a per-pixel loss with an entropy term on half-precision NCHW logits, odd plane size
        dict(name='scores_planes_19_train', op='scores', rows=4, classes=19, inner=769 * 769, last=False, dtype='bf16', top_k=1, train=True, masked=0.0),
        # one tile of a large picture, 512 x 1024: arg-max class with its log probability and the entropy
        dict(name='scores8_512x1024', op='scores8', n=1, h=64, w=128, classes=19, dtype='fp32', top_k=1, train=False),
        # evaluation of a batch of full pictures with three alternatives each
        dict(name='scores8_1024x2048', op='scores8', n=4, h=128, w=256, classes=19, dtype='fp32', top_k=3, train=False),
        # training with a per-pixel loss and an entropy term: eight full pictures, forward and backward
        dict(name='scores8_train', op='scores8', n=8, h=128, w=256, classes=19, dtype='fp32', top_k=0, train=True),
        # the smallest call: the gradients of a classification head, eight tensors
        dict(name='clip_head', op='clip', tensors=8, elements=20011, dtype='fp32'),
        # every parameter of a large network kept in bf16, 400 tensors
        dict(name='clip_400_bf16', op='clip', tensors=400, elements=200_000_003, dtype='bf16'),
        # the gradients of DenseASPP161 before another optimizer's step, 35.4 M elements in 500 tensors
        dict(name='clip_500', op='clip', tensors=500, elements=35_400_000, dtype='fp32'),
        # the optimizer step of DenseASPP161 with clipping: parameters, moments, bf16 copy
        dict(name='adam_161', op='adam', tensors=500, elements=35_400_000, dtype='fp32'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['scores', 'scores', 'scores', 'scores8', 'scores8', 'clip', 'clip', 'adam'])
    if op == 'scores':
        last = rng.random() < 0.5
        dtype = rng.choice(['fp32', 'bf16', 'fp16'])
        train = rng.random() < 0.5
        top_k = rng.choice([0, 1, 2, 3, 5, 8])
        if last:
            classes = _log_int(rng, 9, 21841)
            rows = _log_int(rng, 1, max(2, 33_000_000 // classes))
            return dict(op='scores', rows=rows, classes=classes, inner=1, last=True, dtype=dtype, top_k=top_k, train=train, masked=rng.choice([0.0, 0.15]))
        classes = _log_int(rng, 9, 180)
        rows = rng.randint(1, 4)
        inner = _log_int(rng, 1, max(2, 33_000_000 // (classes * rows)))
        return dict(op='scores', rows=rows, classes=classes, inner=inner, last=False, dtype=dtype, top_k=top_k, train=train, masked=rng.choice([0.0, 0.15]))
    if op == 'scores8':
        h = _log_int(rng, 1, 128)
        w = _log_int(rng, 1, 256)
        n = rng.randint(1, 3)
        return dict(op='scores8', n=n, h=h, w=w, classes=rng.choice([19, 19, rng.randint(9, 32)]), dtype=rng.choice(['fp32', 'fp32', 'bf16', 'fp16']),
                    top_k=rng.choice([0, 1, 2, 3, 5]), train=rng.random() < 0.5)
    if op == 'adam':
        return dict(op='adam', tensors=rng.randint(1, 700), elements=_log_int(rng, 4000, 35_000_000), dtype='fp32')
    dtype = rng.choice(['fp32', 'bf16'])
    return dict(op='clip', tensors=rng.randint(1, 700), elements=_log_int(rng, 4000, 100_000_000), dtype=dtype)


# ------------------------------------------------------------------------------------------------ states
def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) * 7919 + 13)


def _sizes(case):
    """Element counts of the tensors: most are small vectors, a few hold most of the elements."""
    rng = np.random.RandomState((case['tensors'] * 31 + case['elements']) % 65521)
    share = np.exp(rng.normal(0.0, 2.0, case['tensors']))
    sizes = np.maximum(1, np.floor(share / share.sum() * case['elements'])).astype(np.int64)
    return [int(s) for s in sizes]


def _buffer(sizes, dtype, g, scale):
    """One buffer with a tensor of every size, each starting at a multiple of 8 elements; zeros between them."""
    starts = np.concatenate([[0], np.cumsum([(s + 7) // 8 * 8 for s in sizes])]).astype(np.int64)
    total = int(starts[-1])
    flat = torch.randn(total, device='cuda', generator=g).mul_(scale)
    if total > sum(sizes):
        ends = torch.from_numpy(starts[:-1] + np.array(sizes, dtype=np.int64)).cuda()
        rest = torch.from_numpy(starts[1:] - starts[:-1] - np.array(sizes, dtype=np.int64)).cuda()
        gap = torch.repeat_interleave(ends - torch.cumsum(rest, 0) + rest, rest) + torch.arange(int(rest.sum()), device='cuda')
        flat[gap] = 0
    flat = flat.to(dtype)
    return flat, [flat[int(a):int(a) + s] for a, s in zip(starts, sizes)]


def prepare(case, seed):
    g = _generator(seed)
    op = case['op']
    dtype = DTYPES[case['dtype']]
    if op in ('clip', 'adam'):
        sizes = _sizes(case)
        flat, grads = _buffer(sizes, dtype, g, 1e-3)
        norm = 1e-3 * math.sqrt(sum(sizes))
        state = dict(case=case, flat=flat, grads=grads, max_norm=0.5 * norm)
        if op == 'adam':
            n = flat.numel()
            state.update(p=torch.randn(n, device='cuda', generator=g) * 0.05, m=torch.randn(n, device='cuda', generator=g) * 1e-4,
                         v=torch.rand(n, device='cuda', generator=g) * 1e-6, shadow=torch.zeros(n, dtype=torch.bfloat16, device='cuda'))
        return state
    if op == 'scores8':
        shape, rows = (case['n'], case['h'], case['w'], case['classes']), (case['n'], 8 * case['h'], 8 * case['w'])
        z = torch.randn(shape, device='cuda', generator=g) * 3
        logits = z.to(dtype).permute(0, 3, 1, 2)           # the classes are innermost, as the network's classifier leaves them
    elif case['last']:
        rows = (case['rows'],)
        z = torch.randn((case['rows'], case['classes']), device='cuda', generator=g) * 3
        if case['masked']:
            z.masked_fill_(torch.rand(z.shape, device='cuda', generator=g) < case['masked'], -math.inf)
            z.masked_fill_(torch.rand(case['rows'], 1, device='cuda', generator=g) < 0.01, -math.inf)     # rows that see nothing
        logits = z.to(dtype)
    else:
        rows = (case['rows'], case['inner'])
        z = torch.randn((case['rows'], case['classes'], case['inner']), device='cuda', generator=g) * 3
        if case['masked']:
            z.masked_fill_(torch.rand(z.shape, device='cuda', generator=g) < case['masked'], -math.inf)
            z.masked_fill_(torch.rand(case['rows'], 1, case['inner'], device='cuda', generator=g) < 0.01, -math.inf)
        logits = z.to(dtype)
    labels = torch.randint(0, case['classes'], rows, device='cuda', generator=g)
    labels[torch.rand(rows, device='cuda', generator=g) < 0.1] = IGNORE
    state = dict(case=case, logits=logits.requires_grad_(case['train']), labels=labels)
    if case['train']:
        # upstream gradients of a weighted per-pixel loss with an entropy term (and of the best alternative's log probability)
        count = float(labels.numel()) if dtype != torch.float16 else 1.0        # fp16: the loss is scaled up before backward
        state['d_logp'] = -torch.rand(rows, device='cuda', generator=g) / count
        state['d_entropy'] = torch.rand(rows, device='cuda', generator=g) * (0.1 / count)
        if case['top_k']:
            state['d_top'] = torch.randn((rows[0], case['top_k']) + rows[1:], device='cuda', generator=g) * (0.1 / count)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state['case']
    if case['op'] in ('clip', 'adam'):
        return _run_own_grads(state, case) if own else _run_plain_grads(state, case)
    return _run_own_scores(state, case) if own else _run_plain_scores(state, case)


_modules = []


def _package():
    if not _modules:
        import denseASPP  # noqa: F401  (registers the package under its importable name)
        from semantic_segmentation_amd import optim, scores
        _modules.extend((optim, scores))
    return _modules


def _run_own_grads(state, case):
    optim, _ = _package()
    if case['op'] == 'clip':
        state['max_norm'] *= 0.9999             # a threshold that sinks, so that every pass clips
        return dict(norm=optim.clip_grads_(state['grads'], state['max_norm']), grads=state['flat'])
    norm = optim.adam_update_(state['p'], state['flat'], state['m'], state['v'], step=10, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                              weight_decay=1e-4, max_grad_norm=state['max_norm'], shadow=state['shadow'])
    return dict(norm=norm, p=state['p'], m=state['m'], v=state['v'], shadow=state['shadow'])


def _run_own_scores(state, case):
    _, scores = _package()
    s = scores.label_scores(state['logits'], state['labels'], top_k=case['top_k'], ignore_index=IGNORE, upsample=8 if case['op'] == 'scores8' else 1)
    out = dict(logp=s.logp, entropy=s.entropy, top_logp=s.top_logp, top_class=s.top_class)
    if case['train']:
        outs, ups = [s.logp, s.entropy], [state['d_logp'], state['d_entropy']]
        if case['top_k']:
            outs.append(s.top_logp)
            ups.append(state['d_top'])
        out['grad'] = torch.autograd.grad(outs, state['logits'], ups)[0]
    return out


def _run_plain_grads(state, case):
    g = state['flat']
    norm = g.float().square().sum(dtype=torch.float64).sqrt().float()
    if case['op'] == 'clip':
        state['max_norm'] *= 0.9999
        coef = torch.clamp(state['max_norm'] / (norm + EPS), max=1.0)
        g.copy_(g.float() * coef)
        return dict(norm=norm, grads=g)
    coef = torch.clamp(state['max_norm'] / (norm + EPS), max=1.0)
    p, m, v = state['p'], state['m'], state['v']
    d = g * coef + 1e-4 * p
    m.mul_(0.9).add_(d * (1 - 0.9))
    v.mul_(0.999).add_(d * d * (1 - 0.999))
    p.sub_(m / (v.sqrt() / math.sqrt(1 - 0.999 ** 10) + 1e-8) * (1e-3 / (1 - 0.9 ** 10)))
    state['shadow'].copy_(p)
    return dict(norm=norm, p=p, m=m, v=v, shadow=state['shadow'])


def _corners(n, device):
    """Of every output index: the two source indices and the second one's weight (scale 8, align_corners=False)."""
    s = (0.125 * (torch.arange(8 * n, device=device, dtype=torch.float32) + 0.5) - 0.5).clamp(min=0)
    i0 = s.to(torch.int64)
    return i0, (i0 + 1).clamp(max=n - 1), s - i0


def _interpolate(low):
    """N x C x h x w in 32 bits -> N x C x 8h x 8w; every product and every sum is rounded by itself."""
    y0, y1, ly = _corners(low.shape[2], low.device)
    x0, x1, lx = _corners(low.shape[3], low.device)
    across = (1 - lx) * low[..., x0] + lx * low[..., x1]
    ly = ly[:, None]
    return (1 - ly) * across[:, :, y0] + ly * across[:, :, y1]


def _fold_axis(g, n):
    """Adjoint of the interpolation along the last axis: 8n -> n.  Padded by 4 on both sides the outputs fall into n + 1 cells
    of 8 that share their two corners."""
    i0, i1, l1 = _corners(n, g.device)
    a = torch.nn.functional.pad(g * (1 - l1), (4, 4)).unflatten(-1, (n + 1, 8)).sum(-1)
    b = torch.nn.functional.pad(g * l1, (4, 4)).unflatten(-1, (n + 1, 8)).sum(-1)
    low = a[..., 1:] + b[..., :-1]        # pixel i is the first corner of cell i + 1 and the second corner of cell i
    low[..., 0] += a[..., 0]              # on the borders both corners are the border pixel
    low[..., -1] += b[..., -1]
    return low


def _run_plain_scores(state, case):
    with torch.no_grad():
        logits, labels, k = state['logits'].detach(), state['labels'], case['top_k']
        z = logits.float()
        if case['op'] == 'scores8':
            z = _interpolate(z)
        classes = z.shape[1]
        m = z.amax(1, keepdim=True)
        some = torch.isfinite(m)
        shifted = torch.where(some, z - m, -math.inf)
        e = shifted.exp()
        s = e.sum(1, keepdim=True)
        lse = m + s.log()
        log_p = torch.where(some, shifted - s.log(), -math.inf)
        p = torch.where(some, e / s, 0.0)
        p_log_p = torch.where(p > 0, p * log_p, 0.0)
        entropy = -p_log_p.sum(1)
        valid = (labels >= 0) & (labels < classes) & (labels != IGNORE)
        at = torch.where(valid, labels, 0).unsqueeze(1)
        logp = torch.where(valid, log_p.gather(1, at).squeeze(1), 0.0)
        out = dict(logp=logp, entropy=entropy, top_logp=None, top_class=None)
        if k:
            rest = z.clone()
            number = torch.arange(classes, device=z.device).view((1, -1) + (1,) * (z.dim() - 2))
            values, chosen = [], []
            for _ in range(k):
                best = rest.amax(1, keepdim=True)
                first = torch.where(rest == best, number, classes).amin(1, keepdim=True)      # the lowest index of equal ones
                values.append(torch.where(torch.isfinite(best), best - lse, -math.inf))
                chosen.append(torch.where(torch.isfinite(best), first, -1))
                rest.scatter_(1, first, -math.inf)
            out['top_logp'], out['top_class'] = torch.cat(values, 1), torch.cat(chosen, 1)
        if case['train']:
            a = torch.where(valid & some.squeeze(1), state['d_logp'], 0.0).unsqueeze(1)
            total = a
            b = state['d_entropy'].unsqueeze(1)
            if k:
                t = torch.where(out['top_class'] >= 0, state['d_top'], 0.0)
                total = a + t.sum(1, keepdim=True)
            d = -p * total - b * (p_log_p + p * entropy.unsqueeze(1))
            d.scatter_add_(1, at, a)
            if k:
                d.scatter_add_(1, out['top_class'].clamp(min=0), t)
            if case['op'] == 'scores8':
                d = _fold_axis(_fold_axis(d, case['w']).transpose(2, 3), case['h']).transpose(2, 3)
            out['grad'] = d.to(logits.dtype)
        return out


# ------------------------------------------------------------------------------------------------ cost and exact values
def work(case):
    size = {'fp32': 4, 'bf16': 2, 'fp16': 2}[case['dtype']]
    if case['op'] in ('clip', 'adam'):
        n = float(sum(_sizes(case)))
        if case['op'] == 'clip':
            return dict(bytes=2 * n * size, flops=3 * n)
        return dict(bytes=30 * n, flops=17 * n)
    if case['op'] == 'scores8':
        pixels = 64.0 * case['n'] * case['h'] * case['w']
        scores = pixels / 64 * case['classes'] * size
    else:
        pixels = float(case['rows']) * case['inner']
        scores = pixels * case['classes'] * size
    moved = scores + pixels * (8 + 4 + 4 + 12 * case['top_k'])
    per = 8.0 + (3.0 if case['op'] == 'scores8' else 0.0)
    if case['train']:
        moved += scores + pixels * (4 + 4 + 4 * case['top_k'])
        per += 8.0 + (4.0 if case['op'] == 'scores8' else 0.0)
    return dict(bytes=moved, flops=per * pixels * case['classes'])


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] in ('clip', 'adam'):
        g = state['flat'].double()
        norm = torch.linalg.vector_norm(g)
        if case['op'] == 'clip':
            return dict(norm=norm, grads=g * min(1.0, 0.9999 * state['max_norm'] / (float(norm) + EPS)))
        p, m, v = state['p'].double(), state['m'].double(), state['v'].double()
        g = g * min(1.0, state['max_norm'] / (float(norm) + EPS)) + 1e-4 * p
        m = 0.9 * m + 0.1 * g
        v = 0.999 * v + 0.001 * g * g
        p = p - 1e-3 * (m / (1 - 0.9 ** 10)) / ((v / (1 - 0.999 ** 10)).sqrt() + 1e-8)
        return dict(norm=norm, p=p, m=m, v=v, shadow=p.clone())
    k = case['top_k']
    z = state['logits'].detach().double()
    if case['op'] == 'scores8':
        # the interpolation as a matrix of each axis: row o holds the weights that output o gives to the source pixels
        def matrix(n):
            src = np.maximum((np.arange(8 * n) + 0.5) / 8 - 0.5, 0.0)
            lo = np.floor(src).astype(np.int64)
            w = np.zeros((8 * n, n))
            np.add.at(w, (np.arange(8 * n), lo), 1 - (src - lo))
            np.add.at(w, (np.arange(8 * n), np.minimum(lo + 1, n - 1)), src - lo)
            return torch.from_numpy(w).to(z.device)
        my, mx = matrix(case['h']), matrix(case['w'])
        n, c, h, w = z.shape
        z = (z.reshape(-1, w) @ mx.t()).view(n, c, h, 8 * w)
        z = (z.transpose(2, 3).reshape(-1, h) @ my.t()).view(n, c, 8 * w, 8 * h).transpose(2, 3)
    classes = z.shape[1]
    log_p = z - torch.logsumexp(z, 1, keepdim=True)
    empty = torch.isneginf(z).all(1, keepdim=True)
    log_p = log_p.masked_fill(empty, -math.inf)
    p = log_p.exp()
    entropy = torch.special.entr(p).sum(1)
    labels = state['labels']
    wanted = torch.nn.functional.one_hot(torch.where(labels == IGNORE, classes, labels), classes + 1)[..., :classes].movedim(-1, 1) > 0
    logp = torch.where(wanted, log_p, 0.0).sum(1)
    out = dict(logp=logp, entropy=entropy, top_logp=None, top_class=None)
    if k:
        # log probabilities alone: which of two equal ones comes first does not change them
        out['top_logp'] = log_p.sort(1, descending=True).values[:, :k]
    if case['train']:
        take = wanted.double() * state['d_logp'].double().unsqueeze(1)
        if k:
            # the plain order of the classes decides which class each alternative's gradient goes to
            order = torch.sort(z, dim=1, descending=True, stable=True)
            t = torch.where(torch.isfinite(order.values[:, :k]), state['d_top'].double(), 0.0)
            take = take.scatter_add(1, order.indices[:, :k], t)
        take = take.masked_fill(empty, 0.0)
        inner = torch.where(p > 0, log_p + entropy.unsqueeze(1), 0.0)
        d = take - p * take.sum(1, keepdim=True) - state['d_entropy'].double().unsqueeze(1) * p * inner
        if case['op'] == 'scores8':
            d = (d.reshape(-1, 8 * w) @ mx).view(n, c, 8 * h, w)
            d = (d.transpose(2, 3).reshape(-1, 8 * h) @ my).view(n, c, w, h).transpose(2, 3)
        out['grad'] = d
    return out
