"""-m gpu: label_scores (log probabilities of labels, entropy, top alternatives) and its gradient against the definition in 64 bits.
Tolerances: tests/scores_ref.py derives them from the roundings of an fp32 evaluation, element by element."""
import math

import pytest
import torch

import scores_ref as R

pytestmark = pytest.mark.gpu

DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def _label_scores(*a, **k):
    import denseASPP  # noqa: F401
    from semantic_segmentation_amd import label_scores
    return label_scores(*a, **k)


def _make(shape, dtype, layout, seed, mask='none', ints=False):
    """Logits of this logical shape N x C x ... (on the CPU) and a function that lays them out on the GPU."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randint(-3, 4, shape, generator=g).float() if ints else torch.randn(shape, generator=g) * 4
    if mask in ('random', 'rows'):
        z[torch.rand(shape, generator=g) < 0.4] = -math.inf
    if mask == 'rows':
        empty = torch.rand((shape[0], 1) + tuple(shape[2:]), generator=g) < 0.3
        empty.view(-1)[0] = True
        z.masked_fill_(empty, -math.inf)
    if mask == 'lowest':
        z[torch.rand(shape, generator=g) < 0.5] = torch.finfo(dtype).min
        z[0] = torch.finfo(dtype).min                    # rows of nothing else: a uniform distribution
    z = z.to(dtype)
    if mask == 'nan':
        flat = z.view(-1)
        n = flat.numel()
        flat[torch.randint(0, n, (max(1, n // 50),), generator=g)] = math.nan
        flat[torch.randint(0, n, (max(1, n // 50),), generator=g)] = math.inf
        flat[torch.randint(0, n, (max(1, n // 5),), generator=g)] = -math.inf
    rows = (shape[0],) + tuple(shape[2:])
    labels = torch.randint(0, shape[1], rows, generator=g)
    odd = torch.rand(rows, generator=g)
    labels[odd < 0.1] = -100
    labels[(odd >= 0.1) & (odd < 0.15)] = -1
    labels[(odd >= 0.15) & (odd < 0.2)] = shape[1]
    labels[(odd >= 0.2) & (odd < 0.23)] = 2 ** 40
    return z, labels, _place(z, layout)


def _place(z, layout):
    c = z.cuda()
    if layout == 'dense':
        return c
    if layout == 'last':                                  # classes innermost
        return c.movedim(1, -1).contiguous().movedim(-1, 1)
    if layout == 'last_odd':                              # classes innermost, rows padded, start off by one element
        n = c.movedim(1, -1)
        big = torch.full(n.shape[:-1] + (n.shape[-1] + 3,), 7.0, dtype=z.dtype, device='cuda')
        big[..., 1:-2] = n
        return big[..., 1:-2].movedim(-1, 1)
    if layout == 'crop':                                  # a window of a larger picture
        big = torch.full((z.shape[0] + 1, z.shape[1] + 2) + tuple(v + 3 for v in z.shape[2:]), 7.0, dtype=z.dtype, device='cuda')
        at = (slice(1, None), slice(1, -1)) + (slice(1, -2),) * (z.dim() - 2)
        big[at] = c
        return big[at]
    if layout == 'step':                                  # every second pixel
        big = torch.full(tuple(z.shape[:-1]) + (2 * z.shape[-1],), 7.0, dtype=z.dtype, device='cuda')
        big[..., ::2] = c
        return big[..., ::2]
    if layout == 'turned':                                # rows run along the other axis
        return c.transpose(-1, -2).contiguous().transpose(-1, -2)
    raise AssertionError(layout)


def _check(z, labels, logits, top_k, train, ignore_index=-100, entropy=True, g_kind='dense', seed=0):
    terms = z.shape[1]
    r = R.scores(z, labels, top_k, ignore_index, terms)
    if train:
        logits = logits.detach().requires_grad_()
    s = _label_scores(logits, None if labels is None else labels.cuda(), top_k=top_k, ignore_index=ignore_index, entropy=entropy)
    if labels is not None:
        R.agree(s.logp, r['logp'], r['logp_tol'], 'logp')
    else:
        assert s.logp is None
    if entropy:
        R.agree(s.entropy, r['entropy'], r['entropy_tol'], 'entropy')
    else:
        assert s.entropy is None
    if top_k:
        assert torch.equal(s.top_class.cpu(), r['top_class'])
        R.agree(s.top_logp, r['top_logp'], r['top_logp_tol'], 'top_logp')
    else:
        assert s.top_logp is None and s.top_class is None
    if not train:
        return
    g = torch.Generator().manual_seed(seed + 77)
    outs, ups = [], [None, None, None]
    for k, o in enumerate((s.logp, s.entropy, s.top_logp)):
        if o is None or (g_kind == 'logp' and k) or (g_kind == 'entropy' and k != 1) or (g_kind == 'top' and k != 2):
            continue
        u = torch.randn(o.shape, generator=g)
        u[torch.rand(o.shape, generator=g) < 0.2] = 0.0
        u = u.cuda()
        if g_kind == 'one':
            u = torch.tensor(0.37 - 0.2 * k).cuda().expand(o.shape)
        if g_kind == 'strided':
            u = torch.stack((u, u), -1)[..., 0]
        outs.append(o)
        ups[k] = u
    grad, = torch.autograd.grad(outs, logits, [u for u in ups if u is not None])
    want, tol = R.gradient(r, ups[0], ups[1], ups[2], terms)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    R.agree(grad, want, tol, 'gradient', logits.dtype)


# ------------------------------------------------------------------------------------------ against the definition
@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('classes', [1, 2, 7, 8, 9, 19, 64, 65, 150, 1023, 1025])
def test_rows_of_classes(classes, dtype):
    z, labels, logits = _make((37, classes), DT[dtype], 'dense', classes)
    for k in sorted({0, 1, min(3, classes), min(5, classes), min(8, classes)}):
        _check(z, labels, logits, k, True)


@pytest.mark.parametrize('shape', [(4096, 2), (4097, 3), (5000, 9), (4351, 16), (4352, 19), (4353, 32), (4500, 33), (4200, 40), (4100, 63), (4400, 64),
                                   (3, 19, 40, 41), (2, 24, 53, 47)])
@pytest.mark.parametrize('dtype', list(DT))
def test_many_rows_of_few_classes(shape, dtype):
    z, labels, logits = _make(shape, DT[dtype], 'last', shape[1])
    for k in (0, 2):
        _check(z, labels, logits, k, True)
    z, labels, logits = _make(shape, DT[dtype], 'last', shape[1], mask='rows')
    _check(z, labels, logits, min(8, shape[1]), True)


@pytest.mark.parametrize('shape', [(131072, 2), (131073, 3), (131071, 19), (131327, 16), (131100, 19), (131328, 32), (131201, 33), (131400, 63), (3, 19, 210, 211)])
@pytest.mark.parametrize('dtype', list(DT))
def test_rows_enough_for_a_lane_each(shape, dtype):
    z, labels, logits = _make(shape, DT[dtype], 'last', shape[1])
    _check(z, labels, logits, 2, True)
    z, labels, logits = _make(shape, DT[dtype], 'last', shape[1], mask='rows')
    _check(z, labels, logits, 0, True)


@pytest.mark.parametrize('mask', ['random', 'lowest', 'nan'])
def test_masks_in_rows_enough_for_a_lane_each(mask):
    for dtype in DT.values():
        z, labels, logits = _make((131100, 9), dtype, 'dense', 11, mask=mask)
        _check(z, labels, logits, 3, True)


@pytest.mark.parametrize('shape,layout', [((1, 3, 2097155), 'dense'), ((2, 3, 1025, 1031), 'dense'), ((2, 3, 1030, 1040), 'crop'), ((2, 3, 1030, 1040), 'step')])
@pytest.mark.parametrize('dtype', list(DT))
def test_planes_with_several_pixels_per_lane_both_ways(shape, layout, dtype):
    z, labels, logits = _make(shape, DT[dtype], layout, 5)
    _check(z, labels, logits, 1, True)
    z, labels, logits = _make(shape, DT[dtype], layout, 6, mask='nan')
    _check(z, labels, logits, 0, True)


@pytest.mark.parametrize('rows,classes', [(1, 5003), (3, 8193), (2, 21841), (1030, 8195), (1, 4096), (1, 100001), (127, 16385), (128, 16385), (20, 4099)])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_long_rows(rows, classes, dtype):
    z, labels, logits = _make((rows, classes), DT[dtype], 'last_odd', classes)
    _check(z, labels, logits, 5, True)
    _check(z, None, logits, 0, True)


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('classes', [2, 3, 4, 5, 19, 150])
@pytest.mark.parametrize('plane', [(1, 1), (3, 5), (17, 31)])
def test_planes(plane, classes, dtype):
    z, labels, logits = _make((2, classes) + plane, DT[dtype], 'dense', classes + plane[1])
    for k in sorted({0, 1, min(3, classes), min(8, classes)}):
        _check(z, labels, logits, k, True)


@pytest.mark.parametrize('dtype,k', [('fp32', 3), ('bf16', 0), ('fp16', 8), ('bf16', 1)])
@pytest.mark.parametrize('shape', [(1, 9, 524289), (3, 9, 419, 421), (2, 9, 600, 512)])
def test_planes_with_several_pixels_per_lane(shape, dtype, k):
    z, labels, logits = _make(shape, DT[dtype], 'dense', k)
    _check(z, labels, logits, k, True)


@pytest.mark.parametrize('layout', ['dense', 'last', 'last_odd', 'crop', 'step', 'turned'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('shape', [(2, 19, 6, 11), (3, 21, 4, 2, 5), (2, 33, 3, 2, 2, 3)])
def test_layouts(shape, dtype, layout):
    z, labels, logits = _make(shape, DT[dtype], layout, len(shape))
    _check(z, labels, logits, 3, True)
    _check(z, labels, logits, 0, True)


@pytest.mark.parametrize('layout', ['crop', 'step'])
def test_large_planes_in_other_layouts(layout):
    z, labels, logits = _make((2, 5, 513, 521), torch.bfloat16, layout, 3)
    _check(z, labels, logits, 1, True)


@pytest.mark.parametrize('mask', ['random', 'rows', 'lowest', 'nan'])
@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('shape', [(64, 5), (40, 19), (9, 150), (5, 3001), (5, 20001), (2, 7, 9, 5), (1, 3, 530000)])
def test_masks_infinities_and_nan(shape, dtype, mask):
    z, labels, logits = _make(shape, DT[dtype], 'dense', 11, mask=mask)
    _check(z, labels, logits, min(3, shape[1]), True)
    _check(z, labels, logits, 0, True)
    _check(z, labels, logits, 0, True, g_kind='logp')


@pytest.mark.parametrize('shape', [(50, 8), (50, 40), (7, 300), (2, 5000), (3, 30001), (2, 19, 7, 9), (1, 20, 530000)])
@pytest.mark.parametrize('k', [1, 2, 3, 8])
def test_ties_go_to_the_lowest_class(shape, k):
    z, labels, logits = _make(shape, torch.bfloat16, 'dense', k, ints=True)
    _check(z, labels, logits, k, True)


@pytest.mark.parametrize('kind', ['logp', 'entropy', 'top', 'one', 'strided'])
@pytest.mark.parametrize('shape', [(33, 19), (2, 19, 5, 7)])
def test_upstream_gradients(shape, kind):
    z, labels, logits = _make(shape, torch.float32, 'dense', 5)
    _check(z, labels, logits, 4, True, g_kind=kind)


def test_ignore_index_may_be_a_class_and_labels_may_be_absent():
    z, labels, logits = _make((60, 19), torch.float32, 'dense', 6)
    _check(z, labels, logits, 2, True, ignore_index=3)
    _check(z, None, logits, 2, True)
    _check(z, labels, logits, 0, True, entropy=False)


def test_one_pixel_one_class():
    s = _label_scores(torch.tensor([[5.0]]).cuda(), torch.tensor([0]).cuda(), top_k=1)
    assert (s.logp.item(), s.entropy.item(), s.top_logp.item(), s.top_class.item()) == (0.0, 0.0, 0.0, 0)


@pytest.mark.parametrize('shape', [(0, 5), (2, 5, 0), (0, 5, 3, 4)])
def test_no_rows(shape):
    logits = torch.zeros(shape, device='cuda', requires_grad=True)
    s = _label_scores(logits, torch.zeros((shape[0],) + shape[2:], dtype=torch.int64, device='cuda'), top_k=2)
    assert s.logp.shape == (shape[0],) + shape[2:] and s.top_class.shape == (shape[0], 2) + shape[2:]
    s.logp.sum().backward()
    assert logits.grad.shape == shape


def test_broadcast_logits_get_the_summed_gradient():
    z, labels, _ = _make((4, 19, 6), torch.float32, 'dense', 9)
    one = z[:1].cuda().requires_grad_()
    s = _label_scores(one.expand(4, -1, -1), labels.cuda())
    u = torch.randn(s.logp.shape, generator=torch.Generator().manual_seed(1))
    grad, = torch.autograd.grad(s.logp, one, u.cuda())
    r = R.scores(z[:1].expand(4, -1, -1), labels, 0, -100, 19)
    want, tol = R.gradient(r, u, None, None, 19)
    R.agree(grad, want.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 4 * R.U * want.abs().sum(0, keepdim=True), 'broadcast')


def test_gradient_against_differences():
    """Directional differences of the definition in 64 bits.  With the step 1e-4 the quotient is off by its third derivative's part,
    below 1e-8 times the sum of the weights."""
    z, labels, logits = _make((20, 13), torch.float32, 'dense', 21)
    labels = labels.clamp(0, 12)
    g = torch.Generator().manual_seed(3)
    w = [torch.randn(20, generator=g), torch.randn(20, generator=g), torch.randn(20, 2, generator=g)]
    v = torch.randn(20, 13, generator=g).double()

    def f(zz):
        lp = torch.log_softmax(zz, 1)
        ent = -(lp.exp() * lp).sum(1)
        top = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :2]
        return (w[0] * lp.gather(1, labels[:, None])[:, 0] + w[1] * ent + (w[2] * lp.gather(1, top)).sum(1)).sum()

    logits = logits.requires_grad_()
    s = _label_scores(logits, labels.cuda(), top_k=2)
    loss = (s.logp * w[0].cuda()).sum() + (s.entropy * w[1].cuda()).sum() + (s.top_logp * w[2].cuda()).sum()
    grad, = torch.autograd.grad(loss, logits)
    r = R.scores(z, labels, 2, -100, 13)
    _, tol = R.gradient(r, w[0], w[1], w[2], 13)
    h = 1e-4
    quot = (f(z.double() + h * v) - f(z.double() - h * v)) / (2 * h)
    got = (grad.double().cpu() * v).sum()
    weights = sum(x.abs().sum() for x in w)
    lim = (tol * v.abs()).sum() + R.U * (grad.double().cpu().abs() * v.abs()).sum() + 1e-6 * weights
    assert abs(float(got - quot)) <= float(lim)


# ------------------------------------------------------------------------------------------ x8 upsampled
def _check8(z, labels, low, top_k, train, entropy=True, ups_mask=None, ignore_index=-100):
    c = z.shape[1]
    full = R.interpolate(z)
    r = R.scores(full, labels, top_k, ignore_index, c, R=_size(z))
    if train:
        low = low.detach().requires_grad_()
    s = _label_scores(low, None if labels is None else labels.cuda(), top_k=top_k, ignore_index=ignore_index, entropy=entropy, upsample=8)
    if labels is not None:
        R.agree(s.logp, r['logp'], r['logp_tol'], 'logp')
    if entropy:
        R.agree(s.entropy, r['entropy'], r['entropy_tol'], 'entropy')
    if top_k:
        assert torch.equal(s.top_class.cpu(), r['top_class'])
        R.agree(s.top_logp, r['top_logp'], r['top_logp_tol'], 'top_logp')
    if not train:
        return
    g = torch.Generator().manual_seed(5)
    outs, ups = [], [None, None, None]
    for k, o in enumerate((s.logp, s.entropy, s.top_logp)):
        if o is None or (ups_mask is not None and k not in ups_mask):
            continue
        u = torch.randn(o.shape, generator=g)
        u[torch.rand(o.shape, generator=g) < 0.2] = 0.0
        outs.append(o)
        ups[k] = u.cuda()
    grad, = torch.autograd.grad(outs, low, [u for u in ups if u is not None])
    want, tol = R.gradient(r, ups[0], ups[1], ups[2], c)
    # a low-resolution pixel sums up to 8 rows, 8 columns, 4 corners and their clamped copies: fewer than 64 additions in a row,
    # each relative to what it adds; the terms of a pixel before they cancel are at most want's and their own sizes
    p = r['p']
    terms = sum(u.double().cpu().abs().expand(r['empty'].shape) for u in ups[:2] if u is not None) if any(u is not None for u in ups[:2]) else 0
    if ups[2] is not None:
        terms = terms + ups[2].double().cpu().abs().sum(1)
    b = 0 if ups[1] is None else ups[1].double().cpu().abs().unsqueeze(1)
    lpf = torch.where(p > 0, r['lp'], 0.0).abs()
    size = want.abs() + p * (terms.unsqueeze(1) + b * (lpf + r['entropy'].unsqueeze(1)))
    lim = R.adjoint(tol) + 64 * R.U * R.adjoint(size)
    assert grad.dtype == low.dtype and grad.shape == low.shape
    R.agree(grad, R.adjoint(want), lim, 'gradient', low.dtype)


def _size(low):
    """Magnitude of the logits where the short form applies (below 1e5), else 0: the other form is the plain one."""
    big = float(low.detach().float().abs().max())
    return big if big < 1e5 else 0.0


def _make8(shape, dtype, layout, seed, ints=False):
    z, _, low = _make(shape, dtype, layout, seed, ints=ints)
    g = torch.Generator().manual_seed(seed + 1)
    rows = (shape[0], 8 * shape[2], 8 * shape[3])
    labels = torch.randint(0, shape[1], rows, generator=g)
    odd = torch.rand(rows, generator=g)
    labels[odd < 0.1] = -100
    labels[(odd >= 0.1) & (odd < 0.15)] = 255
    return z, labels, low


@pytest.mark.parametrize('hw', [(1, 1), (1, 9), (7, 1), (2, 2), (3, 7), (4, 8), (8, 16), (5, 31), (13, 6)])
@pytest.mark.parametrize('dtype', list(DT))
def test_upsampled_sizes(hw, dtype):
    z, labels, low = _make8((2, 19) + hw, DT[dtype], 'last', hw[0] + hw[1])
    for k in (0, 1, 3, 8):
        _check8(z, labels, low, k, True)


@pytest.mark.parametrize('classes', [1, 2, 7, 8, 9, 16, 17, 19, 24, 25, 32])
def test_upsampled_class_counts(classes):
    z, labels, low = _make8((1, classes, 5, 6), torch.float32, 'dense', classes)
    _check8(z, labels, low, min(2, classes), True)
    _check8(z, labels, low, 0, True, ups_mask=(0,))
    _check8(z, None, low, 0, True)


@pytest.mark.parametrize('layout', ['dense', 'last', 'last_odd', 'crop', 'step', 'turned'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_upsampled_layouts(layout, dtype):
    z, labels, low = _make8((3, 11, 5, 9), DT[dtype], layout, 2)
    _check8(z, labels, low, 2, True)


@pytest.mark.parametrize('ups', [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_upsampled_upstream_gradients(ups):
    z, labels, low = _make8((2, 19, 4, 6), torch.float32, 'last', 8)
    _check8(z, labels, low, 3, True, ups_mask=ups)


def test_upsampled_ties_and_lowest_values():
    z, labels, low = _make8((2, 19, 4, 5), torch.float32, 'last', 4, ints=True)
    _check8(z, labels, low, 4, True)
    z[:, 3:] = -1e30                                   # finite masks
    _check8(z, labels, _place(z, 'last'), 3, True)


@pytest.mark.parametrize('classes', [5, 19, 30])
@pytest.mark.parametrize('depth', [100.0, 3000.0, 1e10, 1e19, 3e20])
def test_upsampled_rows_that_peak_at_different_classes(depth, classes):
    """Neighbouring pixels hundreds of units (and far more) apart in opposite classes: between them every class is far below either
    peak."""
    z, labels, low = _make8((1, classes, 4, 6), torch.float32, 'last', 7)
    z = (z - depth)
    z[:, 0, ::2, ::2] += depth
    z[:, 1, 1::2, ::2] += depth
    z[:, 2, ::2, 1::2] += depth
    z[:, 3, 1::2, 1::2] += depth
    _check8(z, labels, _place(z, 'last'), 3, True)
    _check8(z, labels, _place(z, 'last'), 0, True)


@pytest.mark.parametrize('x', [2, 3, 7, 8, 12, 15, 16])
def test_upsampled_steep_pixels_beside_ordinary_ones(x):
    """One steep column of pixels: the short form holds for some waves only, and the two passes, whose waves hold different columns, do
    not agree about all of them."""
    z, labels, _ = _make8((1, 19, 6, 20), torch.float32, 'last', 7)
    z[:, :, :, x] -= 200.0
    z[:, 0, ::2, x] += 200.0
    z[:, 1, 1::2, x] += 200.0
    for layout in ('last', 'dense'):
        _check8(z, labels, _place(z, layout), 2, True)
        _check8(z, labels, _place(z, layout), 0, True)


@pytest.mark.parametrize('x', [7, 8, 9])
def test_upsampled_far_pixels_beside_ordinary_ones(x):
    """Logits of 1e6 in a few pixels: what lies two pixels away has the gradient it has without them.  Each of the two gradients is off by
    15 R half-steps in an exponent (short form), R = 20 bounding the ordinary logits, relative to the sizes of its terms."""
    z, labels, _ = _make8((1, 19, 6, 20), torch.float32, 'last', 9)
    z = z.clamp(-20, 20)
    g = torch.Generator().manual_seed(1)
    u = [torch.randn(1, 48, 160, generator=g) for _ in range(2)]
    grads = []
    for far in (False, True):
        t = z.clone()
        if far:
            t[:, ::3, :, x] = 1.0e6
        low = _place(t, 'last').requires_grad_()
        s = _label_scores(low, labels.cuda(), upsample=8)
        grad, = torch.autograd.grad((s.logp, s.entropy), low, [v.cuda() for v in u])
        grads.append(grad.double().cpu()[..., :x - 1])
    r = R.scores(R.interpolate(z), labels, 0, -100, 19, R=20.0)
    size = r['p'] * (u[0].abs().double().unsqueeze(1) + u[1].abs().double().unsqueeze(1) * (r['lp'].abs() + r['entropy'].unsqueeze(1)))
    lim = (2 * 15 * 20 + 64) * R.U * R.adjoint(size)[..., :x - 1] + 2 * 64 * R.U * R.adjoint(u[0].abs().double().unsqueeze(1).expand_as(size))[..., :x - 1]
    assert bool(((grads[0] - grads[1]).abs() <= lim).all())


@pytest.mark.parametrize('k', [2, 3, 8])
def test_upsampled_near_ties(k):
    """Classes that differ in their last bits alone, in both directions, and both zeros."""
    g = torch.Generator().manual_seed(k)
    base = torch.randn(1, 1, 5, 6, generator=g).expand(1, 19, 5, 6)
    z = base * (1 + torch.randint(-3, 4, (1, 19, 5, 6), generator=g) * 2.0 ** -23)
    z = torch.where(torch.rand(1, 1, 5, 6, generator=g) < 0.2, torch.randn(1, 19, 5, 6, generator=g).sign() * 0.0, z)
    labels = torch.randint(0, 19, (1, 40, 48), generator=g)
    _check8(z, labels, _place(z, 'last'), k, True)


def test_upsampled_nan_stays_where_it_is_read():
    z, labels, low = _make8((1, 19, 6, 7), torch.float32, 'last', 4)
    z[0, 5, 2, 3] = math.nan
    low = _place(z, 'last').requires_grad_()
    s = _label_scores(low, labels.cuda(), top_k=1, upsample=8)
    bad = torch.isnan(R.interpolate(z)).any(1)
    assert bad.any() and not bad.all()
    assert torch.equal(torch.isnan(s.entropy).cpu(), bad) and torch.equal((s.top_class[:, 0] == -1).cpu(), bad)
    # nothing flows back from those pixels: the gradient is finite everywhere
    u = torch.where(bad.cuda(), 0.0, 1.0)
    grad, = torch.autograd.grad((s.logp, s.entropy), low, (u, u))
    assert torch.isfinite(grad).all() and grad.abs().sum() > 0


# ------------------------------------------------------------------------------------------ streams, graphs, repetition
def _both(logits, labels, k, upsample):
    s = _label_scores(logits, labels, top_k=k, upsample=upsample)
    loss = s.logp.sum() + 0.1 * s.entropy.sum() + (s.top_logp * 0.3).sum()
    grad, = torch.autograd.grad(loss, logits)
    return tuple(t.detach() for t in (*s, grad))          # keeps no graph of the leaf alive


CASES = [((64, 1203), 1), ((2, 19, 61, 33), 1), ((2, 19, 9, 11), 8)]


@pytest.mark.parametrize('shape,upsample', CASES)
def test_same_bits_every_time_and_on_two_streams(shape, upsample):
    mk = _make8 if upsample == 8 else _make
    z, labels, logits = mk(shape, torch.float32, 'dense', 3)
    labels, logits = labels.cuda(), logits.requires_grad_()
    first = _both(logits, labels, 2, upsample)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for rep in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                results.append(_both(logits, labels, 2, upsample))
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


@pytest.mark.parametrize('shape,upsample', CASES)
def test_captured_and_replayed(shape, upsample):
    mk = _make8 if upsample == 8 else _make
    sets = [mk(shape, torch.bfloat16, 'dense', s) for s in (1, 2, 3)]
    logits = torch.empty_like(sets[0][2]).requires_grad_()
    labels = sets[0][1].cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _both(logits, labels, 2, upsample)                 # warm-up
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs over the same tensors share no workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _both(logits, labels, 2, upsample)
        graphs.append((graph, out))
    for z, lab, src in sets:
        with torch.no_grad():
            logits.copy_(src)
            labels.copy_(lab.cuda())
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, out in graphs]
        fresh = src.clone().requires_grad_()
        want = _both(fresh, lab.cuda(), 2, upsample)
        torch.cuda.synchronize()
        for g in got:
            for a, b in zip(g, want):
                assert torch.equal(a, b)


def test_capture_beside_a_live_graph_of_the_same_leaf_is_refused(monkeypatch):
    """The accumulator of a leaf belongs to the stream of the graph that made it: asked whether that is seen, without a real capture."""
    leaf = torch.randn(4, 5, device='cuda', requires_grad=True)
    alive = _label_scores(leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.ones(4, device='cuda')
        want, = torch.autograd.grad(_label_scores(leaf).entropy, leaf, g)
        s = _label_scores(leaf)
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
            with pytest.raises(RuntimeError, match='captured'):
                torch.autograd.grad(s.entropy, leaf, g)
            del alive, s
            got, = torch.autograd.grad(_label_scores(leaf).entropy, leaf, g)       # the side stream's own graph
            twice = leaf * 2.0
            torch.autograd.grad(_label_scores(twice).entropy, twice, g)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_views_that_are_negated_when_read():
    z = torch.randn(6, 19, 5, 4, device='cuda')
    labels = torch.randint(0, 19, (6, 5, 4), device='cuda')
    a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
    s, t = _label_scores(torch._neg_view(a), torch._neg_view(-labels), top_k=2), _label_scores(-b, labels, top_k=2)
    for x, y in zip(s, t):
        assert torch.equal(x, y)
    g = torch.randn(6, 5, 4, device='cuda')
    s.logp.backward(torch._neg_view(g))
    t.logp.backward(-g)
    assert torch.equal(a.grad, b.grad)


def test_more_rows_than_a_grid_has_lanes():
    """2^32 + 300 rows of 2 classes (17 GB): a lane per row no longer is one launch."""
    n = 2 ** 32 + 300
    logits = torch.zeros((n, 2), dtype=torch.bfloat16, device='cuda')
    logits[-3:] = torch.tensor([[1.0, -1.0], [0.5, 0.0], [-math.inf, -math.inf]], dtype=torch.bfloat16)
    logits.requires_grad_()
    s = _label_scores(logits)
    g = torch.ones((), device='cuda').expand(n)
    grad, = torch.autograd.grad(s.entropy, logits, g)
    with torch.no_grad():
        flat = s.entropy[:-3]
        assert abs(float(flat.min()) - math.log(2)) < 1e-6 and float(flat.max()) == float(flat.min())
        assert not bool(grad[:-3].any()) and not bool(grad[-1].any())
        tail = logits[-3:].detach().cpu().double()
        p = torch.softmax(tail[:2], 1)
        h = -(p * p.log()).sum(1)
        assert torch.allclose(s.entropy[-3:-1].cpu().double(), h, rtol=0, atol=8 * R.U)
        assert float(s.entropy[-1]) == 0.0
        want = -p * (p.log() + h[:, None])
        assert torch.allclose(grad[-3:-1].cpu().double(), want, rtol=2.0 ** -8, atol=8 * R.U)


def test_second_derivative_is_refused():
    logits = torch.randn(4, 5, device='cuda', requires_grad=True)
    s = _label_scores(logits)
    g, = torch.autograd.grad(s.entropy.sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_overwritten_logits_are_noticed():
    leaf = torch.randn(4, 5, device='cuda', requires_grad=True)
    logits = leaf * 1.0
    s = _label_scores(logits)
    logits.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        s.entropy.sum().backward()


# ------------------------------------------------------------------------------------------ the network's own path
def _tiny(train, dtype=torch.bfloat16):
    from e2e_common import TINY_CFG, make_pair
    ref, mod = make_pair(TINY_CFG)
    mod.set_compute_dtype(dtype)
    mod = mod.cuda()
    mod.train(train)
    ref.train(train)
    return ref, mod


def test_network_scores_are_those_of_its_logits():
    from e2e_common import make_batch
    _, mod = _tiny(False)
    x, labels = make_batch(2, 64, 96)
    s = mod.score(x.cuda(), labels.cuda(), top_k=3)
    low = mod.forward_lowres(x.cuda())
    full = R.interpolate(low)
    r = R.scores(full, labels, 3, 255, 19, R=_size(low))
    R.agree(s.logp, r['logp'], r['logp_tol'], 'logp')
    R.agree(s.entropy, r['entropy'], r['entropy_tol'], 'entropy')
    assert torch.equal(s.top_class.cpu(), r['top_class'])
    R.agree(s.top_logp, r['top_logp'], r['top_logp_tol'], 'top_logp')
    # the mean of the labelled pixels is the loss of the reference's criterion on model(x)
    count = (labels != 255).sum()
    loss = torch.nn.functional.cross_entropy(mod(x.cuda()), labels.cuda(), ignore_index=255)
    assert abs(float(-s.logp.sum() / count) - float(loss)) <= 1e-5 * float(loss)
    assert mod.score(x.cuda(), entropy=False, top_k=1).logp is None


def test_training_through_scores_matches_the_oracle():
    """A weighted per-pixel loss with an entropy term, through the network in its fp32 form, against torch autograd on the oracle:
    gradients to 1e-3, the bound of the fp32 form's gradient tests."""
    from e2e_common import grad_report, make_batch, make_dropout_masks
    ref, mod = _tiny(True, torch.float32)
    x, labels = make_batch(2, 64, 96)
    masks = make_dropout_masks(ref, 2, torch.Generator().manual_seed(5))
    weight = torch.rand(labels.shape, generator=torch.Generator().manual_seed(6))
    n = labels.numel()
    out = torch.log_softmax(ref(x, masks), 1)
    valid = labels != 255
    logp = torch.where(valid, out.gather(1, torch.where(valid, labels, 0).unsqueeze(1)).squeeze(1), 0.0)
    loss_r = -(logp * weight).sum() / n + 0.1 * (-(out.exp() * out).sum(1)).mean() - 0.05 * out.amax(1).mean()
    loss_r.backward()
    s = mod.score(x.cuda(), labels.cuda(), top_k=1, dropout_masks={k: v.cuda() for k, v in masks.items()})
    loss = -(s.logp * weight.cuda()).sum() / n + 0.1 * s.entropy.mean() - 0.05 * s.top_logp.mean()
    loss.backward()
    assert abs(float(loss.detach()) - float(loss_r.detach())) <= 1e-4 * abs(float(loss_r.detach()))
    rel, cos, worst = grad_report({k: p.grad for k, p in ref.named_parameters()}, {k: p.grad.cpu() for k, p in mod.named_parameters()})
    assert rel <= 1e-3, (rel, cos, worst)


def test_scores_of_a_training_step_agree_with_its_fused_loss():
    """Loss and low-resolution gradient of train_step against label_scores on the same logits (one forward pass: BatchNorm's sums are
    atomic and make no two passes alike).  Both gradients are fp32 evaluations of one formula: each within the bound of the definition."""
    from e2e_common import make_batch
    _, mod = _tiny(True)
    x, labels = make_batch(2, 64, 96)
    loss = float(mod.train_step(x.cuda(), labels.cuda(), generator=torch.Generator(device='cuda').manual_seed(3)).detach())
    eng = mod.engine(2, 64, 96)
    low = eng.low_logits().clone().requires_grad_()
    dlow = eng.dlogits.view(2, 8, 12, 32)[..., :19].permute(0, 3, 1, 2).cpu().double()
    count = (labels != 255).sum().item()
    s = _label_scores(low, labels.cuda(), ignore_index=255, upsample=8)
    mine = -s.logp.sum() / count
    assert abs(float(mine.detach()) - loss) <= 64 * R.U * loss                 # two sums of 1e4 terms of one sign, trees of fewer than 64 roundings
    grad, = torch.autograd.grad(mine, low)
    r = R.scores(R.interpolate(low), labels, 0, 255, 19, R=_size(low))
    u = torch.full(labels.shape, -1.0 / count)
    want, tol = R.gradient(r, u, None, None, 19)
    lim = 2 * (R.adjoint(tol) + 64 * R.U * R.adjoint(want.abs() + r['p'] / count))
    R.agree(grad, R.adjoint(want), lim / 2, 'gradient')
    R.agree(grad, dlow, lim, 'fused loss')


def test_image_gradient_flows_through_score():
    from e2e_common import make_batch
    _, mod = _tiny(True)
    x, labels = make_batch(1, 64, 64)
    xg = x.cuda().requires_grad_()
    (-mod.score(xg, labels.cuda(), generator=torch.Generator(device='cuda').manual_seed(3)).logp.mean()).backward()
    assert xg.grad.shape == x.shape and torch.isfinite(xg.grad).all() and xg.grad.abs().sum() > 0


def test_stale_pass_is_refused():
    from e2e_common import make_batch
    _, mod = _tiny(True)
    x, labels = make_batch(1, 64, 64)
    first = mod.score(x.cuda(), labels.cuda())
    mod.score(x.cuda(), labels.cuda())
    with pytest.raises(RuntimeError, match='another pass'):
        first.logp.sum().backward()
    s = mod.score(x.cuda(), labels.cuda())
    s.logp.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match='another pass'):
        s.logp.sum().backward()


def test_score_backward_clip_and_update_together():
    """A step of one's own: scores of the network, a loss, its backward pass, the clipped Adam update; and clipping in place beside it.
    The first Adam step is lr g / (|g| + eps) with the clipped g: 16 half-steps of it and one of the parameter."""
    from e2e_common import make_batch
    from semantic_segmentation_amd.optim import FusedAdam, clip_grad_norm_
    _, mod = _tiny(True, torch.float32)
    x, labels = make_batch(2, 64, 96)
    opt = FusedAdam(mod, lr=1e-3)
    s = mod.score(x.cuda(), labels.cuda(), top_k=2)
    (-s.logp.mean() + 0.1 * s.entropy.mean()).backward()
    params = list(mod.parameters())
    g = [p.grad.double().cpu() for p in params]
    before = [p.detach().double().cpu() for p in params]
    want = math.sqrt(sum(float(t.square().sum()) for t in g))
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for c, p in zip(copies, params):
        c.grad = p.grad.clone()
    limit = 0.5 * want
    coef = limit / (want + 1e-6)
    norm = clip_grad_norm_(copies, limit)
    assert abs(float(norm) - want) <= 1.01 * R.U * want
    for c, t in zip(copies, g):
        R.agree(c.grad, t * coef, 3 * R.U * (t * coef).abs(), 'clipped')
    norm = opt.step(max_grad_norm=limit)
    assert abs(float(norm) - want) <= 1.01 * R.U * want
    for p, b, t in zip(params, before, g):
        step = 1e-3 * (t * coef) / ((t * coef).abs() + 1e-8)
        R.agree(p.detach(), b - step, 16 * R.U * step.abs() + R.U * b.abs(), 'parameter')
    after = mod.score(x.cuda(), labels.cuda())
    assert bool(torch.isfinite(after.logp).all())
