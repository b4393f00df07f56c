"""The class scores and their gradient in 64 bits, from their definition, with the rounding errors the fp32 kernels may make."""
import torch

U = 2.0 ** -24          # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # spacing below the normal range


def scores(z, labels, top_k, ignore_index, terms, R=0.0):
    """z: N x C x ... any float type; everything returned in float64 / int64, with absolute tolerances.  `terms`: additions that
    one running sum of the kernel may hold in a row.

    With d = z - m (one rounding, relative U), e = exp(d) is off by at most (2|d| + 2) U, so s = sum e by (terms + 2 + 2 sum p|d|) U, and
    sum p|d| = H - log s <= H.  t = sum d e likewise, relative to sum |d| e = s (H - log s).  log adds 2 U (1 + log s), log s <= H.

    R > 0: the x8 form on logits of magnitude up to R, which takes each exponential from the one of the row above.  Its logarithm is off by
    delta = 15 R U (the reference's own interpolation included) + 23 U (7 steps of 3 U, the first exponential); d is counted from a
    reference up to 2 R off the maximum, so that log s and t / s are 2 R larger before they cancel."""
    zd = z.detach().double().cpu()
    c = zd.shape[1]
    bad = (torch.isnan(zd) | torch.isposinf(zd)).any(1)
    empty = torch.isneginf(zd).all(1)
    m = torch.where(empty | bad, 0.0, zd.nan_to_num(nan=0.0, posinf=0.0).amax(1))
    d = zd - m.unsqueeze(1)
    e = d.exp()
    s = e.sum(1)
    log_s = s.log()
    lp = torch.where(empty.unsqueeze(1), -float('inf'), d - log_s.unsqueeze(1))
    p = torch.where(empty.unsqueeze(1), 0.0, e / s.unsqueeze(1))
    h = torch.where(p > 0, -p * lp, 0.0).sum(1)
    h = torch.where(bad, float('nan'), h)
    hh = torch.where(bad, 0.0, h)
    out = dict(p=p, lp=lp, entropy=h, empty=empty, bad=bad)
    delta = 15 * R * U + 23 * U if R else 0.0
    out['delta'], out['shift'] = delta, 2.0 * R
    out['entropy_tol'] = U * (2 * terms + 16) * (1 + hh) + 2 * delta * (1 + 2 * hh) + (terms + 8) * U * 2 * R
    base = U * ((terms + 8) * (1 + hh) + 4 * hh) + 2 * delta + 8 * U * R
    if labels is not None:
        lab = labels.cpu()
        has = (lab != ignore_index) & (lab >= 0) & (lab < c)
        at = torch.where(has, lab, 0).unsqueeze(1)
        v = lp.gather(1, at).squeeze(1)
        v = torch.where(bad, float('nan'), v)
        out['has'] = has
        out['at'] = at
        out['logp'] = torch.where(has, v, 0.0)
        out['logp_tol'] = base + 4 * U * out['logp'].abs().nan_to_num(posinf=0.0)
    if top_k:
        zt = z.detach().float().cpu()
        order = torch.sort(zt.nan_to_num(nan=-float('inf'), posinf=-float('inf'), neginf=-float('inf')), dim=1, descending=True, stable=True)
        idx = order.indices[:, :top_k]
        val = lp.gather(1, idx)
        gone = torch.isneginf(zd.gather(1, idx)) | empty.unsqueeze(1)
        val = torch.where(gone, -float('inf'), val)
        idx = torch.where(gone, -1, idx)
        out['top_class'] = torch.where(bad.unsqueeze(1), -1, idx)
        out['top_logp'] = torch.where(bad.unsqueeze(1), float('nan'), val)
        out['top_logp_tol'] = base.unsqueeze(1) + 4 * U * out['top_logp'].abs().nan_to_num(posinf=0.0)
    return out


def gradient(r, g_logp, g_entropy, g_top, terms):
    """dz of the scores `r` and its absolute tolerance (before the rounding to the result's type).  p is off by (terms + 8 + 4 |lp|) U,
    the bracket by a few roundings of its terms."""
    p, lp = r['p'], r['lp']
    rows = r['empty'].shape
    zero = torch.zeros(rows, dtype=torch.float64)
    a = zero if g_logp is None else torch.where(r['has'], g_logp.double().cpu().expand(rows), 0.0)
    b = zero if g_entropy is None else g_entropy.double().cpu().expand(rows)
    A = a.clone()
    delta = torch.zeros_like(p)
    size = a.abs()
    alive = (a != 0) | (b != 0)
    if g_logp is not None:
        delta.scatter_add_(1, r['at'], a.unsqueeze(1))
    if g_top is not None:
        idx = r['top_class']
        raw = g_top.double().cpu().expand(idx.shape)
        t = torch.where(idx >= 0, raw, 0.0)
        alive = alive | torch.where(r['bad'].unsqueeze(1), raw != 0, t != 0).any(1)
        A = A + t.sum(1)
        size = size + t.abs().sum(1)
        delta.scatter_add_(1, idx.clamp(min=0), t)
    h = torch.where(r['bad'], 0.0, r['entropy'])
    lpf = torch.where(p > 0, lp, 0.0)
    spread = lpf + h.unsqueeze(1)
    g = delta - p * (A.unsqueeze(1) + b.unsqueeze(1) * spread)
    g = torch.where(r['bad'].unsqueeze(1), float('nan'), g)
    alive = (alive & ~r['empty']).unsqueeze(1)
    g = torch.where(alive, g, 0.0)
    inner = size.unsqueeze(1) + b.abs().unsqueeze(1) * (lpf.abs() + h.unsqueeze(1))
    tol = U * ((terms + 16 + 4 * lpf.abs()) * p * inner + (terms + 16) * b.abs().unsqueeze(1) * p * (1 + h.unsqueeze(1)) + 4 * delta.abs() + 10 * size.unsqueeze(1) * (delta != 0))
    more = 2 * r['delta'] * p * inner + b.abs().unsqueeze(1) * p * (2 * r['delta'] + (terms + 8) * U * r['shift'])
    tol = torch.where(alive & ~r['bad'].unsqueeze(1), tol + more, 0.0)
    return g, tol


def agree(got, want, tol, what, dtype=torch.float32):
    """Same non-finite values in the same places, the rest within tol plus half a step of `dtype`."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ': NaN in other places'
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what + ': infinities in other places'
    lim = (tol.expand(want.shape) + half_step(dtype) * want.abs() + tiny(dtype))[fin]
    err = (got - want)[fin].abs()
    if err.numel():
        worst = (err / lim).max().item()
        assert worst <= 1.0, '%s: error %.3g times its bound' % (what, worst)


def corners(n):
    s = (0.125 * (torch.arange(8 * n, dtype=torch.float32) + 0.5) - 0.5).clamp(min=0)
    i0 = s.to(torch.int64)
    return i0, (i0 + 1).clamp(max=n - 1), s - i0


def interpolate(low):
    """The x8 upsample in fp32 with every product and sum rounded by itself (torch's elementwise kernels do not contract)."""
    low = low.detach().float().cpu()
    y0, y1, ly = corners(low.shape[2])
    x0, x1, lx = corners(low.shape[3])
    r = (1 - lx) * low[..., x0] + lx * low[..., x1]
    ly = ly.unsqueeze(1)
    return (1 - ly) * r[:, :, y0] + ly * r[:, :, y1]


def adjoint(g):
    """Adjoint of the x8 upsample in 64 bits, by the weight matrix of each axis."""
    def matrix(n):
        i0, i1, l1 = corners(n)
        w = torch.zeros(8 * n, n, dtype=torch.float64)
        w.index_put_((torch.arange(8 * n), i0), 1 - l1.double(), accumulate=True)
        w.index_put_((torch.arange(8 * n), i1), l1.double(), accumulate=True)
        return w
    h, w = g.shape[2] // 8, g.shape[3] // 8
    return torch.matmul(torch.matmul(matrix(h).t().contiguous(), g), matrix(w))
