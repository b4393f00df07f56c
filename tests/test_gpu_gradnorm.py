"""-m gpu: global gradient norm, clipping and the clipped Adam update against their formulas in 64 bits.  The sums are fp64, so a norm is
off by its rounding to fp32 (2^-24) alone; a clipped gradient by the rounding of the coefficient, of the product (2^-24 each) and of
its own type."""
import math

import pytest
import torch

import scores_ref as R

pytestmark = pytest.mark.gpu
U = R.U
F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16


def _optim():
    import denseASPP  # noqa: F401
    from semantic_segmentation_amd import optim
    return optim


def _tensors(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(sizes)]


def _norm(ts, kind=2.0):
    if kind == 2.0:
        return math.sqrt(sum(float(t.detach().cpu().double().square().sum()) for t in ts))
    return max(float(t.detach().cpu().double().abs().max()) for t in ts if t.numel())


def _near(got, want):
    assert got.dtype == F32 and got.dim() == 0
    assert abs(float(got) - want) <= 1.01 * U * want, (float(got), want)


def _check_clip(ts, max_norm, kind=2.0, fn=None):
    before = [t.detach().cpu().double() for t in ts]
    want = _norm(ts, kind)
    got = (fn or _optim().clip_grads_)(ts, max_norm, norm_type=kind)
    _near(got, want)
    coef = min(1.0, max_norm / (want + 1e-6))
    for t, b in zip(ts, before):
        if coef == 1.0:
            assert torch.equal(t.cpu().double(), b)
        else:
            R.agree(t, b * coef, 3 * U * (b * coef).abs(), 'clipped', t.dtype)


SIZES = [1, 2, 3, 7, 8, 9, 255, 256, 1000, 8191, 8192, 8193, 16385, 100003]


@pytest.mark.parametrize('dtypes', [(F32,), (B16,), (F16,), (F32, B16, F16)])
@pytest.mark.parametrize('kind', [2.0, math.inf])
def test_sizes_and_types(dtypes, kind):
    ts = _tensors(SIZES, dtypes, 1)
    _near(_optim().grad_norm(ts, kind), _norm(ts, kind))
    _check_clip(ts, 0.25 * _norm(ts, kind), kind)


@pytest.mark.parametrize('sizes', [[1], [8192], [8193], [1, 2, 3, 4, 5, 6, 7], [1000] * 8, [1000] * 9, [4096, 4096], [4096, 4097]])
@pytest.mark.parametrize('dtypes', [(F32,), (B16,), (F16, F32)])
@pytest.mark.parametrize('kind', [2.0, math.inf])
def test_few_elements(sizes, dtypes, kind):
    ts = _tensors(sizes, dtypes, sum(sizes))
    _check_clip(ts, 0.3 * _norm(ts, kind), kind)
    _check_clip(ts, 2.0 * _norm(ts, kind), kind)


@pytest.mark.parametrize('n', [1, 5, 8192, 8193, 3_000_001])
@pytest.mark.parametrize('dtype', [F32, B16])
def test_one_tensor(n, dtype):
    t, = _tensors([n], (dtype,), n)
    _near(_optim().grad_norm(t), _norm([t]))
    _check_clip([t], 0.5)


@pytest.mark.parametrize('count', [179, 399, 400, 401, 1300])
def test_many_tensors(count):
    ts = _tensors([(i * 37) % 501 + 1 for i in range(count)], (F32, F32, B16), count)
    _check_clip(ts, 1.0)


def test_ranges_longer_than_one_entry_and_launches_longer_than_their_chunks():
    """3e8 elements: longer than one range of a launch, followed by enough to pass the 65535 chunks of one launch; an odd start between."""
    buf = torch.ones(300_000_007, dtype=B16, device='cuda')
    more = torch.ones(280_000_001, dtype=B16, device='cuda')
    ts = [buf[1:], more, torch.full((5,), 2.0, device='cuda')]
    want = math.sqrt(300_000_006 + 280_000_001 + 20)
    _near(_optim().grad_norm(ts), want)
    _near(_optim().clip_grads_(ts, 0.5 * want), want)
    half = torch.tensor(0.5 * want / (want + 1e-6)).to(B16)
    assert bool((ts[0] == half.cuda()).all()) and bool((ts[1] == half.cuda()).all())
    assert float(buf[0]) == 1.0 and abs(float(ts[2][4]) - 1.0) < 1e-5


def test_more_blocks_than_one_launch_keeps():
    ts = _tensors([20_000_000, 5, 30_000_001], (F32, B16), 3, 1e-3)
    _check_clip(ts, 1.0)


def test_not_exceeded_leaves_every_bit():
    ts = _tensors(SIZES, (F32, B16, F16), 2)
    _check_clip(ts, 2.0 * _norm(ts))
    _check_clip(ts, math.inf)


def test_max_norm_zero():
    ts = _tensors([100, 9], (F32,), 2)
    _optim().clip_grads_(ts, 0.0)
    assert all(float(t.abs().max()) == 0.0 for t in ts)


@pytest.mark.parametrize('scale', [1e30, 1e-30, 1e-41])
def test_magnitudes_whose_squares_leave_fp32(scale):
    ts = [t * 1.0 for t in _tensors([1000, 77], (F32,), 4, scale)]
    want = _norm(ts)
    got = _optim().grad_norm(ts)
    assert abs(float(got) - want) <= 1.01 * U * want + 2.0 ** -150
    if scale > 1:
        _check_clip(ts, 1.0)


def test_unaligned_and_permuted_and_strided():
    g = torch.Generator().manual_seed(5)
    for dt in (F32, B16, F16):
        buf = torch.randn(5000, generator=g).to(dt).cuda()
        conv = torch.randn(24, 3, 3, 16, generator=g).to(dt).cuda().permute(0, 3, 1, 2)          # channels_last, as the arena's views
        wide = torch.randn(40, 33, generator=g).to(dt).cuda()
        box = torch.randn(6, 7, 8, generator=g).to(dt).cuda()
        rest_w, rest_b = wide[:, 20:].clone(), buf[2000:].clone()
        ts = [buf[1:1000], buf[1001:2000], conv, wide[:, 3:20], box[::2, 1:, ::3].transpose(0, 2), buf[:0]]
        rest_box = box.clone()
        _check_clip(ts, 3.0)
        assert torch.equal(wide[:, 20:], rest_w) and torch.equal(buf[2000:], rest_b)          # what lies between is left as it was
        kept = torch.ones_like(box, dtype=torch.bool)
        kept[::2, 1:, ::3] = False
        assert torch.equal(box[kept], rest_box[kept])


def test_expanded_counts_every_element():
    t = torch.tensor([2.0, 3.0]).cuda().unsqueeze(1).expand(2, 10)
    _near(_optim().grad_norm([t]), math.sqrt(10 * (4 + 9)))


@pytest.mark.parametrize('value', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('kind', [2.0, math.inf])
def test_nonfinite(value, kind):
    optim = _optim()
    ts = _tensors([1000, 9], (F32, B16), 6)
    ts[0][777] = value
    keep = [t.clone() for t in ts]
    with pytest.raises(RuntimeError, match='not finite'):
        optim.clip_grads_(ts, 1.0, kind, error_if_nonfinite=True)
    for t, k in zip(ts, keep):
        assert torch.equal(t.nan_to_num(nan=5.0), k.nan_to_num(nan=5.0))
    norm = optim.clip_grads_(ts, 1.0, kind)
    if math.isnan(value):
        assert math.isnan(float(norm)) and all(torch.isnan(t).all() for t in ts)
    else:                               # coefficient 0: the infinite entry becomes NaN, as in torch
        assert math.isinf(float(norm)) and torch.isnan(ts[0][777])
        ts[0][777] = 0.0
        assert all(float(t.abs().max()) == 0.0 for t in ts)


def test_parameters_like_torch():
    optim = _optim()
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.Flatten(), torch.nn.Linear(8 * 36, 5), torch.nn.Linear(5, 2)).cuda()
    net(torch.randn(4, 3, 8, 8, device='cuda'))[:, 0].sum().backward()
    extra = torch.nn.Parameter(torch.zeros(3, device='cuda'))                    # has no gradient
    params = list(net.parameters()) + [extra]
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for a, b in zip(params, twin):
        b.grad = None if a.grad is None else a.grad.clone()
    version = params[0].grad._version
    got = optim.clip_grad_norm_(params, 0.1)
    want = torch.nn.utils.clip_grad_norm_(twin, 0.1)
    # torch's own fp32 norm of 1500 values: a tree of norms, fewer than 32 roundings deep
    assert abs(float(got) - float(want)) <= 32 * U * float(want)
    for a, b in zip(params, twin):
        assert (a.grad is None) == (b.grad is None)
        if a.grad is not None:
            R.agree(a.grad, b.grad.double().cpu(), 40 * U * b.grad.double().cpu().abs(), 'grad')
    assert params[0].grad._version > version
    assert float(optim.clip_grad_norm_([extra], 1.0)) == 0.0
    assert float(optim.clip_grad_norm_(iter([]), 1.0)) == 0.0


def test_refusals():
    optim = _optim()
    a = torch.ones(10, device='cuda')
    with pytest.raises(ValueError, match='share memory'):
        optim.clip_grads_([a, a], 1.0)
    with pytest.raises(ValueError, match='share memory'):
        optim.clip_grads_([a[:6], a[5:]], 1.0)
    with pytest.raises(ValueError, match='share memory'):
        optim.clip_grads_([torch.ones(1, device='cuda').expand(4)], 1.0)
    with pytest.raises(ValueError, match='norm_type'):
        optim.clip_grads_([a], 1.0, norm_type=1)
    with pytest.raises(ValueError, match='max_norm'):
        optim.clip_grads_([a], -1.0)
    with pytest.raises(ValueError, match='max_norm'):
        optim.clip_grads_([a], math.nan)
    with pytest.raises(TypeError, match='float64'):
        optim.grad_norm([a.double()])
    with pytest.raises(ValueError, match='GPU'):
        optim.grad_norm([a.cpu()])
    with pytest.raises(ValueError, match='GPU'):
        optim.grad_norm([a, a.cpu()])
    with pytest.raises(ValueError, match='requires grad'):
        optim.clip_grads_([a.clone().requires_grad_()], 1.0)
    with pytest.raises(ValueError, match='contiguous'):
        optim.grad_norm([torch.ones(200_000, device='cuda')[::2]])
    assert torch.equal(a, torch.ones_like(a))
    p, m, v = a.clone(), a.clone(), a.clone()
    with pytest.raises(ValueError, match='share memory'):
        optim.adam_update_(a, a, m, v, 1)
    with pytest.raises(ValueError, match='step'):
        optim.adam_update_(p, a, m, v, 0)
    with pytest.raises(ValueError, match='one size'):
        optim.adam_update_(p, a[:5], m, v, 1)
    with pytest.raises(ValueError, match='shadow'):
        optim.adam_update_(p, a, m, v, 1, shadow=torch.zeros(10, device='cuda'))
    with pytest.raises(ValueError, match='max_grad_norm'):
        optim.adam_update_(p, a, m, v, 1, max_grad_norm=-2.0)
    with pytest.raises(ValueError, match='grad_scale'):
        optim.adam_update_(p, a, m, v, 1, grad_scale=0.0)


def test_same_bits_and_two_streams_and_replay():
    optim = _optim()
    ts = _tensors(SIZES, (F32, B16), 9)
    first = optim.grad_norm(ts)
    for _ in range(3):
        assert torch.equal(optim.grad_norm(ts), first)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = optim.grad_norm(ts)
    here = optim.grad_norm(ts)
    torch.cuda.synchronize()
    assert torch.equal(other, first) and torch.equal(here, first)
    static = [torch.empty_like(t) for t in ts]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = optim.clip_grads_(static, 2.0)
    for seed in (1, 2, 3):
        src = _tensors(SIZES, (F32, B16), seed, seed)
        for a, b in zip(static, src):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got, got_norm = [t.clone() for t in static], norm.clone()
        want_norm = optim.clip_grads_(src, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(got_norm, want_norm)
        for a, b in zip(got, src):
            assert torch.equal(a, b)


@pytest.mark.parametrize('n', [1, 3, 4, 1027, 1_000_003])
@pytest.mark.parametrize('scale,max_norm', [(1.0, 0.5), (0.125, 0.01), (0.5, math.inf)])
def test_adam_update(n, scale, max_norm):
    optim = _optim()
    g = torch.Generator().manual_seed(n)
    grad = torch.randn(n, generator=g)
    p, m, v = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.1, torch.rand(n, generator=g) * 0.1
    dev = [t.cuda() for t in (p, grad, m, v)]
    shadow = torch.zeros(n, dtype=B16, device='cuda')
    norm = optim.adam_update_(dev[0], dev[1], dev[2], dev[3], 7, lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, grad_scale=scale,
                              max_grad_norm=max_norm, shadow=shadow)
    want = scale * _norm([grad])
    _near(norm, want)
    coef = min(1.0, max_norm / (want + 1e-6)) if math.isfinite(max_norm) else 1.0
    gd, pd, md, vd = grad.double() * scale * coef, p.double(), m.double(), v.double()
    gp = gd + 1e-2 * pd
    gsize = gd.abs() + 1e-2 * pd.abs()                    # 4 roundings of the terms of g
    m2, v2 = 0.9 * md + 0.1 * gp, 0.999 * vd + 0.001 * gp * gp
    m_tol = U * (4 * 0.9 * md.abs() + 8 * 0.1 * gsize)
    v_tol = U * (4 * 0.999 * vd + 16 * 0.001 * gsize * gp.abs())
    R.agree(dev[2], m2, m_tol, 'm')
    R.agree(dev[3], v2, v_tol, 'v')
    den = (v2 / (1 - 0.999 ** 7)).sqrt() + 1e-8
    step = 2e-3 / (1 - 0.9 ** 7) * m2 / den
    # sqrt halves v's relative error; division, factor and difference round once each
    p_tol = 2e-3 / (1 - 0.9 ** 7) * m_tol / den + step.abs() * (0.5 * v_tol / v2 + 10 * U) + U * pd.abs()
    R.agree(dev[0], pd - step, p_tol, 'p')
    assert torch.equal(dev[1].cpu(), grad)                # the gradient is read only
    assert torch.equal(shadow, dev[0].to(B16))


def test_fused_adam_clips_and_reports_the_norm():
    """score -> loss -> backward -> clipped step, as a training loop has them; the update is checked against the formula on the
    gradients that the network itself produced."""
    from e2e_common import TINY_CFG, make_batch, make_pair
    optim = _optim()
    _, mod = make_pair(TINY_CFG)
    mod = mod.cuda().train()
    opt = optim.FusedAdam(mod, lr=1e-3, weight_decay=1e-4)
    x, labels = make_batch(2, 64, 96)
    gen = torch.Generator(device='cuda').manual_seed(1)
    for step in (1, 2, 3):
        for p in mod.parameters():
            p.grad = None
        s = mod.score(x.cuda(), labels.cuda(), generator=gen)
        (-s.logp.mean() + 0.1 * s.entropy.mean()).backward()
        grads = [p.grad.clone() for p in mod.parameters()]
        want = _norm(grads)
        before = [p.detach().cpu().double() for p in mod.parameters()]
        norm = opt.step(max_grad_norm=0.3 * want)
        _near(norm, want)
        if step == 1:
            coef = 0.3 * want / (want + 1e-6)
            for p, b, g in zip(mod.parameters(), before, grads):
                gp = coef * g.cpu().double() + 1e-4 * b
                size = (coef * g.cpu().double()).abs() + 1e-4 * b.abs()
                gt = 8 * U * size
                den = gp.abs() + 1e-8
                # p - lr g / (|g| + eps): d/dg of g/(|g| + eps) = eps / (|g| + eps)^2, largest within the tolerance of g
                near = (gp.abs() - gt).clamp(min=0) + 1e-8
                tol = 1e-3 * (1e-8 * gt / near ** 2).clamp(max=2.0) + 1e-3 * 32 * U + U * b.abs()
                R.agree(p, b - 1e-3 * gp / den, tol, 'p')
        assert torch.isfinite(mod._flat).all()
        assert torch.equal(mod._w16, mod._flat.to(B16))
    assert opt.step_count == 3


def test_clipping_counts_the_pending_scale_of_a_reducer():
    from e2e_common import TINY_CFG, make_batch, make_pair
    optim = _optim()
    _, mod = make_pair(TINY_CFG)
    mod = mod.cuda().train()
    opt = optim.FusedAdam(mod)
    x, labels = make_batch(1, 64, 64)
    mod.train_step(x.cuda(), labels.cuda())
    want = _norm([mod._gflat])
    mod._grad_scale = 0.25
    _near(opt.step(max_grad_norm=1e9), 0.25 * want)
    assert mod._grad_scale == 1.0
    before = mod._flat.clone()
    with pytest.raises(ValueError, match='max_grad_norm'):
        opt.step(max_grad_norm=math.nan)
    with pytest.raises(ValueError, match='scale'):
        opt.step(grad_scale=0.0, max_grad_norm=1.0)
    assert opt.step_count == 1 and torch.equal(before, mod._flat)


def test_unclipped_step_agrees_with_the_plain_one():
    """max_grad_norm=inf against step(): the plain kernel forms 1 - beta from fp32 betas (1.3e-5 relative at 0.999), nothing else differs."""
    from e2e_common import TINY_CFG, make_batch, make_pair
    optim = _optim()
    mods = []
    for clip in (None, math.inf):
        _, mod = make_pair(TINY_CFG)
        mod = mod.cuda().train()
        opt = optim.FusedAdam(mod, lr=1e-3)
        x, labels = make_batch(1, 64, 64)
        torch.manual_seed(4)
        mod.train_step(x.cuda(), labels.cuda(), generator=torch.Generator(device='cuda').manual_seed(2))
        if mods:
            mod._gflat.copy_(mods[0][1])
        else:
            grads = mod._gflat.clone()
        assert (opt.step(max_grad_norm=clip) is None) == (clip is None)
        mods.append((mod._flat.clone(), grads))
    assert float((mods[0][0] - mods[1][0]).abs().max()) <= 1e-3 * 2e-5 + 2 * U * float(mods[0][0].abs().max())
