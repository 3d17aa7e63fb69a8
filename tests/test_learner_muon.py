"""CPU side of the orthogonalised updates (drloco_amd.muon, dl_orth_update): refusals of the C and of the Python entry points, workspace
sizes, the optimiser's bookkeeping.  Nothing here touches a device."""
import ctypes as C
import math
import os

import pytest
import torch

from drloco_amd import learner_lib as ll
from drloco_amd import lib, muon


@pytest.fixture(scope='module')
def L():
    if not os.path.exists(ll.LIB_PATH):
        ll.build()
    return ll.load()


def shape(batch=1, rows=8, cols=16, **kw):
    s = ll.OrthShape(batch=batch, rows=rows, cols=cols, a=3.0, b=-4.0, c=2.0, beta=0.9, weight_keep=1.0, gain=1.0, steps=5)
    for n in ('grad', 'momentum', 'momentum_out', 'weight', 'out'):
        setattr(s, n + '_b', rows * cols), setattr(s, n + '_r', cols)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


BAD = [dict(grad_type=3), dict(weight_type=-1), dict(out_type=7), dict(reserved=1), dict(batch=-1), dict(rows=-1), dict(cols=-1), dict(batch=65536), dict(rows=(1 << 20) + 1), dict(cols=1 << 30),
       dict(rows=1 << 20, cols=1 << 13), dict(steps=0), dict(steps=101), dict(steps=-5)] + [{f'{n}_{a}': -1} for n in ('grad', 'momentum', 'momentum_out', 'weight', 'out') for a in 'br']


@pytest.mark.parametrize('bad', BAD, ids=str)
def test_bad_shapes_are_refused(L, bad):
    s, p = C.byref(shape(**bad)), 4096
    assert L.dl_orth_workspace_bytes(s) == -1
    assert L.dl_orth_update(s, p, None, None, None, p, p, None) == -1
    assert len(L.dl_learner_last_error()) > 5


def test_bad_pointers_are_refused(L):
    s, p = C.byref(shape(1, 80, 90)), 4096          # (a size that needs a workspace)
    assert L.dl_orth_workspace_bytes(None) == -1
    assert L.dl_orth_update(None, p, None, None, None, p, p, None) == -1
    for k in (0, 4, 5):
        a = [p, None, None, None, p, p, None]
        a[k] = None
        assert L.dl_orth_update(s, *a) == -1
    assert L.dl_orth_update(s, p, p, None, None, p, p, None) == -1
    assert L.dl_orth_update(s, p, None, p, None, p, p, None) == -1
    assert L.dl_orth_update(s, p, None, None, None, p, p + 4, None) == -1


def test_empty_shapes_are_done_at_once(L):
    for kw in (dict(batch=0), dict(rows=0), dict(cols=0)):
        s = C.byref(shape(**kw))
        assert L.dl_orth_workspace_bytes(s) == 0 and L.dl_orth_update(s, None, None, None, None, None, None, None) == 0


@pytest.mark.parametrize('batch,rows,cols', [(1, 1, 1), (1, 8, 512), (3, 512, 512), (1, 4096, 8192), (7, 1031, 4099)])
def test_the_workspace_is_a_small_multiple_of_the_matrix(L, batch, rows, cols):
    size = L.dl_orth_workspace_bytes(C.byref(shape(batch, rows, cols)))
    up = lambda n: -(-n // 128) * 128
    m, n = sorted((up(rows), up(cols)))
    # three X, A and Q in four bytes an element, up to 1024 partial sums of squares a matrix, split sums of 4 KB for 512 workgroups at most
    assert 0 <= size <= batch * (3 * m * n * 4 + 2 * m * m * 4 + 8192) + 512 * 4096 + 4096


z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize('args,kw,error', [
    ((z(8),), {}, ValueError), ((z(2, 2, dtype=torch.float64),), {}, TypeError), (([1.0],), {}, TypeError), ((z(2, 2), 0), {}, ValueError), ((z(2, 2), 101), {}, ValueError),
    ((z(2, 2), 2.5), {}, ValueError), ((z(2, 2), 5, (1.0, 2.0)), {}, ValueError), ((z(2, 2), 5, (1.0, 2.0, math.inf)), {}, ValueError), ((z(2, 2),), {}, lib.DrlocoError),
])
def test_refusals_of_orthogonalise(args, kw, error):
    with pytest.raises(error):
        muon.orthogonalise(*args, **kw)


@pytest.mark.parametrize('args,kw,error', [
    ((z(4, 2), z(2, 4), z(4, 2)), {}, ValueError), ((z(4, 2), z(4, 2), z(4, 3)), {}, ValueError), ((z(4, 2), z(4, 2), z(4, 2, dtype=torch.bfloat16)), {}, TypeError),
    ((z(4), z(4), z(4)), {}, ValueError), ((z(4, 2), z(4, 2), z(4, 2)), dict(steps=0), ValueError), ((z(4, 2), z(4, 2), z(4, 2)), {}, lib.DrlocoError),
])
def test_refusals_of_the_update(args, kw, error):
    with pytest.raises(error):
        muon.muon_update(*args, lr=0.1, **kw)


def test_destinations_are_looked_at():
    w, other = z(6, 4), z(7, 4)
    ok = lambda t, aliases: muon._result('f', 'out', t, w, torch.float32, aliases)
    assert ok(w, [(True, w)]) is w and ok(z(6, 4), [(False, w)]) is not None
    for t, aliases in ((w, [(False, w)]), (other[1:], [(True, other[:6])]), (z(4, 6).t(), []), (z(6, 5), []), (z(6, 4, dtype=torch.float16), [])):
        with pytest.raises(ValueError):
            ok(t, aliases)


def test_the_optimiser_refuses_what_is_not_a_matrix():
    p = lambda *s, **kw: torch.nn.Parameter(z(*s, **kw))
    for bad in (p(8), p(4, 4, dtype=torch.float64), torch.nn.Parameter(z(4, 6).t())):
        with pytest.raises(ValueError):
            muon.HipMuon([p(4, 4), bad])
    for kw in (dict(lr=-1.0), dict(beta=1.0), dict(weight_decay=-0.1), dict(steps=0), dict(lr=math.nan)):
        with pytest.raises(ValueError):
            muon.HipMuon([p(4, 4)], **kw)
    opt = muon.HipMuon([p(4, 4)])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[p(3)]))
    assert len(opt.param_groups) == 1 and opt.step() is None          # (no gradients: nothing to do)


def test_the_optimiser_state_round_trips_in_32_bits():
    q = torch.nn.Parameter(z(4, 4, dtype=torch.bfloat16))
    a, b = muon.HipMuon([q]), muon.HipMuon([q], lr=0.5)
    a.state[q]['momentum'] = torch.full((4, 4), 1.0 + 2.0 ** -20)
    b.load_state_dict(a.state_dict())
    m = b.state[q]['momentum']
    assert m.dtype == torch.float32 and torch.equal(m, a.state[q]['momentum']) and m.data_ptr() != a.state[q]['momentum'].data_ptr()
    assert b.param_groups[0]['lr'] == 0.02


def test_a_first_step_is_not_captured(monkeypatch):
    p = torch.nn.Parameter(torch.ones(4, 5))
    p.grad = torch.ones(4, 5)
    opt = muon.HipMuon([p])
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='before it is captured'):
        opt.step()
    assert not opt.state[p]


def grows(steps, a, b, c):
    """The largest |s|, s^2 and |q(s^2)| over singular values 0 .. 1 on a fine grid, before each of the steps."""
    import numpy as np
    s, most = np.linspace(0.0, 1.0, 200001), 0.0
    for _ in range(steps):
        q = a + b * s ** 2 + c * s ** 4
        with np.errstate(over='ignore', invalid='ignore'):
            most = max(most, np.abs(s).max(), (s ** 2).max(), np.abs(q).max())
        # (every value up to the largest may be a singular value)
        s = np.linspace(0.0, np.abs(s * q).max(), 200001)
        if not most < 1e6:
            return 1e6
    return most


COEFS = [(5, muon.COEFFICIENTS), (100, muon.COEFFICIENTS), (5, muon.CUBIC), (100, muon.CUBIC), (1, (59.9, 0.0, 0.0)), (1, (60.1, 0.0, 0.0)), (1, (64.0, -64.0, 0.0)), (1, (1.0, -61.5, 0.0)), (1, (0.0, 100.0, -100.0)),
         (1, (0.0, 300.0, -300.0)), (2, (7.7, 0.0, 0.0)), (2, (7.8, 0.0, 0.0)), (5, (3.0, -4.0, 2.0)), (4, (3.0, -4.0, 2.0)), (3, (8.287, -23.596, 17.3)), (5, (2.0, -1.5, 0.5)), (1, (0.0, 0.0, 0.0)),
         (1, (1e300, 1.0, 1.0)), (2, (1.0, 1e200, -1e200)), (5, (1.875, -1.25, 0.375)), (7, (0.0, 0.0, 1.0)), (3, (-3.4445, 4.775, -2.0315))]


@pytest.mark.parametrize('steps,coefficients', COEFS, ids=str)
def test_coefficients_that_leave_the_range_are_refused(L, steps, coefficients):
    """float16 planes times 2^10 end at 63.97: what grows to 60 is refused, by the C entry points and the Python ones alike"""
    fits = grows(steps, *coefficients) < 60
    a, b, c = coefficients
    assert L.dl_orth_check_coefficients(steps, a, b, c) == (0 if fits else -1)
    s = shape(steps=steps, a=a, b=b, c=c)
    assert L.dl_orth_update(C.byref(s), None, None, None, None, None, None, None) == -1
    assert (b'coefficients' in L.dl_learner_last_error()) == (not fits)
    make = lambda: muon.HipMuon([torch.nn.Parameter(z(4, 4))], steps=steps, coefficients=coefficients)
    if fits:
        make()
        with pytest.raises(lib.DrlocoError):          # (nothing wrong but the device)
            muon.orthogonalise(z(2, 2), steps, coefficients)
    else:
        for call in (make, lambda: muon.orthogonalise(z(2, 2), steps, coefficients), lambda: muon.muon_update(z(2, 2), z(2, 2), z(2, 2), lr=0.1, steps=steps, coefficients=coefficients)):
            with pytest.raises(ValueError):
                call()


def test_coefficients_that_are_no_numbers_are_refused(L):
    for bad in (math.nan, math.inf, -math.inf):
        for k in range(3):
            cs = [1.5, -0.5, 0.1]
            cs[k] = bad
            assert L.dl_orth_check_coefficients(1, *cs) == -1
    assert L.dl_orth_check_coefficients(0, 1.5, -0.5, 0.0) == -1 and L.dl_orth_check_coefficients(101, 1.5, -0.5, 0.0) == -1
