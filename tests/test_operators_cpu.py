"""Refusals of the class-score and gradient-norm entry points that need no GPU: the C ABI's checks of descriptors, and the Python
side's checks of arguments."""
import ctypes
import math

import pytest
import torch

import denseASPP  # noqa: F401
from semantic_segmentation_amd import DenseASPP, _lib, label_scores, optim

GOOD = 0x10000          # never read: the checks come before any launch


def _err():
    return _lib.load().dsaspp_last_error().decode()


def _scores(**k):
    d = _lib.scores_desc()
    f = dict(dtype=1, n_class=19, d0=2, d1=1, d2=8, s0=152, s1=0, s2=1, sc=8, logits=GOOD, labels=GOOD, ignore_index=255, logp=GOOD)
    f.update(k)
    for n, v in f.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize('bad,message', [
    (dict(dtype=3), 'dtype'), (dict(dtype=-1), 'dtype'), (dict(n_class=0), 'n_class'), (dict(top_k=9, top_logp=GOOD, top_class=GOOD), 'top_k'),
    (dict(n_class=4, top_k=5, top_logp=GOOD, top_class=GOOD), 'top_k'), (dict(top_k=-1), 'top_k'), (dict(d2=0), 'row counts'),
    (dict(d0=1 << 39, d1=4), 'row counts'), (dict(s2=-1), 'stride'), (dict(logits=None), 'null logits'), (dict(logits=GOOD + 2), 'aligned'),
    (dict(labels=None), 'labels'), (dict(top_k=2), 'top_logp'), (dict(logp=None), 'nothing')])
def test_scores_forward_descriptor(bad, message):
    assert _lib.load().dsaspp_scores_fwd(ctypes.byref(_scores(**bad)), None) != 0
    assert message in _err()


@pytest.mark.parametrize('bad,message', [
    (dict(), 'stats'), (dict(stats=GOOD, dlogits=GOOD), 'upstream'), (dict(stats=GOOD, dlogits=GOOD, g_logp=GOOD, labels=None), 'labels'),
    (dict(stats=GOOD, dlogits=GOOD, g_entropy=GOOD), 'entropy'), (dict(stats=GOOD, dlogits=GOOD, g_top=GOOD), 'top_class'),
    (dict(stats=GOOD, dlogits=GOOD + 1, g_logp=GOOD), 'aligned')])
def test_scores_backward_descriptor(bad, message):
    assert _lib.load().dsaspp_scores_bwd(ctypes.byref(_scores(**bad)), None) != 0
    assert message in _err()


def test_scores_workspace_for_few_long_rows():
    lib = _lib.load()
    assert lib.dsaspp_scores_workspace(ctypes.byref(_scores())) == 0
    long = dict(n_class=50000, d0=2, d2=1, s0=50000, sc=1)
    need = lib.dsaspp_scores_workspace(ctypes.byref(_scores(**long)))
    assert need > 0 and need % 2 == 0
    assert lib.dsaspp_scores_workspace(ctypes.byref(_scores(**dict(long, d0=1000)))) == 0
    assert lib.dsaspp_scores_fwd(ctypes.byref(_scores(**long, ws=GOOD, ws_len=need - 1)), None) != 0
    assert 'workspace' in _err()
    assert lib.dsaspp_scores_workspace(ctypes.byref(_scores(dtype=9))) == -1


def _scores8(**k):
    d = _lib.scores8_desc()
    f = dict(n_img=1, h=4, w=5, n_class=19, dtype=1, g_dtype=1, sn=380, sy=95, sx=19, sc=1, logits=GOOD, labels=GOOD, ignore_index=255, logp=GOOD)
    f.update(k)
    for n, v in f.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize('bad,message', [
    (dict(n_class=33), 'n_class'), (dict(h=0), 'geometry'), (dict(w=1 << 20), 'geometry'), (dict(n_img=1 << 30, h=1000, w=1000), 'too many'),
    (dict(n_img=1 << 24, h=1, w=1), 'too many'),
    (dict(top_k=9), 'top_k'), (dict(logits=GOOD + 1), 'aligned'), (dict(sx=-1), 'stride'), (dict(labels=None), 'labels'), (dict(logp=None), 'nothing')])
def test_scores8_forward_descriptor(bad, message):
    assert _lib.load().dsaspp_scores8_fwd(ctypes.byref(_scores8(**bad)), None) != 0
    assert message in _err()


def test_scores8_backward_descriptor():
    lib = _lib.load()
    need = lib.dsaspp_scores8_workspace(ctypes.byref(_scores8()))
    assert need == 1 * 1 * 2 * 45 * 19                       # one tile of cells across (6 of 8), two down (5 of 8), 9 x 5 corner pixels each
    assert lib.dsaspp_scores8_workspace(ctypes.byref(_scores8(n_class=40))) == -1
    full = dict(g_logp=GOOD, stats=GOOD, dlogits=GOOD, gn=380, gy=95, gx=19, gc=1, ws=GOOD, ws_len=need)
    for bad, message in ((dict(ws_len=need - 1), 'workspace'), (dict(ws=None), 'workspace'), (dict(gx=0), 'gradient strides'), (dict(dlogits=None), 'dlogits'),
                         (dict(g_dtype=7), 'g_dtype'), (dict(g_logp=None), 'upstream'), (dict(g_top=GOOD), 'top_class'), (dict(stats=None), 'stats'),
                         (dict(g_entropy=GOOD), 'entropy of the forward')):
        assert lib.dsaspp_scores8_bwd(ctypes.byref(_scores8(**dict(full, **bad))), None) != 0
        assert message in _err(), message


def _clip(ranges, **k):
    arr = (_lib.grad_range * max(1, len(ranges)))()
    for r, (p, n, dt) in zip(arr, ranges):
        r.p, r.n, r.dtype = p, n, dt
    d = _lib.clip_desc()
    d.ranges, d.n_ranges, d.norm_type, d.scale, d.max_norm = ctypes.cast(arr, ctypes.c_void_p), len(ranges), 2, 1.0, 1.0
    d.ws, d.ws_len, d.norm = GOOD, 1 << 20, GOOD
    for n, v in k.items():
        setattr(d, n, v)
    return d, arr


@pytest.mark.parametrize('ranges,bad,message', [
    ([(GOOD, 8, 3)], {}, 'dtype'), ([(GOOD, 0, 1)], {}, 'empty'), ([(None, 8, 1)], {}, 'null'), ([(GOOD + 2, 8, 1)], {}, 'aligned'),
    ([(GOOD, 8, 1)], dict(norm_type=1), 'norm_type'), ([(GOOD, 8, 1)], dict(scale=0.0), 'scale'), ([(GOOD, 8, 1)], dict(scale=math.inf), 'scale'),
    ([(GOOD, 8, 1)], dict(ws_len=0), 'workspace'), ([(GOOD, 8, 1)], dict(ws=None), 'workspace'), ([(GOOD, 8, 1)], dict(max_norm=-1.0), 'max_norm'),
    ([(GOOD, 8, 1)], dict(scale=0.5), 'scale must be 1'), ([(GOOD, 8, 1)], dict(norm=None), 'null output')])
def test_clip_descriptor(ranges, bad, message):
    d, keep = _clip(ranges, **bad)
    assert _lib.load().dsaspp_clip_scale(ctypes.byref(d), None) != 0
    assert message in _err()


def test_norm_workspace_sizes():
    lib = _lib.load()
    assert lib.dsaspp_grad_norm_workspace(ctypes.byref(_clip([])[0])) == 0
    small, k1 = _clip([(GOOD, 8192, 1), (GOOD, 1, 1)])
    big, k2 = _clip([(GOOD, 1 << 33, 1)])
    assert 1 <= lib.dsaspp_grad_norm_workspace(ctypes.byref(small)) <= lib.dsaspp_grad_norm_workspace(ctypes.byref(big))
    bad, k3 = _clip([(GOOD, -1, 1)])
    assert lib.dsaspp_grad_norm_workspace(ctypes.byref(bad)) == -1


def test_adam_clipped_descriptor():
    lib = _lib.load()
    c, keep = _clip([(GOOD, 8, 1)])
    a = _lib.adam_clip_desc()
    assert lib.dsaspp_adam_step_clipped(ctypes.byref(a), ctypes.byref(c), None) != 0
    assert 'positive' in _err()
    a.n, a.p, a.g, a.m, a.v, a.step = 8, GOOD, GOOD, GOOD, GOOD + 1, 1
    assert lib.dsaspp_adam_step_clipped(ctypes.byref(a), ctypes.byref(c), None) != 0
    assert 'aligned' in _err()


def test_python_refusals():
    z = torch.zeros(2, 5)
    with pytest.raises(ValueError, match='GPU'):
        label_scores(z)
    with pytest.raises(TypeError, match='float64'):
        label_scores(z.double())
    with pytest.raises(TypeError, match='list'):
        label_scores([1.0])
    with pytest.raises(ValueError, match='GPU'):
        optim.grad_norm([z])
    with pytest.raises(ValueError, match='GPU'):
        optim.clip_grads_([z], 1.0)
    assert float(optim.grad_norm([])) == 0.0


def test_shape_checks():
    """The checks behind label_scores and DenseASPP.score; device and shapes are all they look at."""
    def check(shape, labels=None, top_k=0, entropy=True, upsample=1):
        _lib.binding().check_scores(shape, 'cuda:0', labels, top_k, entropy, upsample)

    for kw, message in ((dict(shape=[5]), 'N x C'), (dict(shape=[2, 3, 4], upsample=8), 'N x C x h x w'), (dict(shape=[2, 33, 4, 4], upsample=8), 'at most 32'),
                        (dict(shape=[2, 0]), 'classes'), (dict(shape=[2, 5], top_k=6), 'top_k'), (dict(shape=[2, 50], top_k=9), 'top_k'),
                        (dict(shape=[2, 5], top_k=-1), 'top_k'), (dict(shape=[2, 5], entropy=False), 'nothing'), (dict(shape=[2, 5], upsample=4), 'upsample'),
                        (dict(shape=[2, 5], labels=torch.zeros(2, dtype=torch.int64)), 'labels'), (dict(shape=[2, 5], labels=torch.zeros(3, dtype=torch.int64)), 'labels')):
        with pytest.raises(ValueError, match=message):
            check(**kw)
    check([2, 5], top_k=5)


def test_row_dimensions_merge():
    rows = _lib.binding().rows_of
    assert rows(torch.zeros(2, 19, 6, 7)) == [(2, 798), (1, 0), (42, 1)]
    assert rows(torch.zeros(2, 6, 7, 19).movedim(-1, 1)) == [(2, 798), (1, 0), (42, 19)]
    assert rows(torch.zeros(2, 19, 8, 9)[:, :, 1:7, 1:8]) == [(2, 1368), (6, 9), (7, 1)]
    assert rows(torch.zeros(2, 5, 4, 5, 6)[:, :, :3, :4, :5]) is None
    assert rows(torch.zeros(7, 19)) == [(7, 19), (1, 0), (1, 0)]


def test_dense_pieces():
    ranges = _lib.binding().ranges_of
    t = torch.zeros(4, 10)
    base = t.data_ptr()
    assert ranges(t[:, 2:5]) == [(base + 4 * (10 * r + 2), 3) for r in range(4)]
    assert ranges(t.t()) == [(base, 40)]
    assert ranges(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))[0][1] == 120
    one = torch.zeros(2, 1).expand(2, 3)
    assert sorted(ranges(one)) == [(one.data_ptr(), 2)] * 3
    box = torch.zeros(3, 4, 5)
    cut = box[::2, 1:3, ::2]
    want = sorted(box.data_ptr() + 4 * int(i) for i in torch.arange(60).view(3, 4, 5)[::2, 1:3, ::2].reshape(-1))
    assert sorted(p for p, n in ranges(cut)) == want and all(n == 1 for _, n in ranges(cut))
    with pytest.raises(ValueError, match='contiguous'):
        ranges(torch.zeros(200_000)[::2])


def test_binding_was_built_from_this_tree():
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location('dsaspp_build', os.path.join(_lib.HERE, 'build.py'))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert _lib.binding().source_hash() == mod.binding_hash() == mod.built_binding_hash()


def test_score_needs_a_gpu_and_multiples_of_eight():
    from conftest import TINY_CFG
    mod = DenseASPP(TINY_CFG)
    with pytest.raises(ValueError, match='multiples of 8'):
        mod.score(torch.zeros(1, 3, 60, 64))
    with pytest.raises(ValueError, match='GPU'):
        mod.score(torch.zeros(1, 3, 64, 64))
    with pytest.raises(ValueError, match='N x 3'):
        mod.score(torch.zeros(1, 4, 64, 64))
