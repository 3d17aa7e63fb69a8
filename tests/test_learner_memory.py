"""CPU side of the gated memory (drloco_amd.memory, include/drloco_learner.h): the library's symbols, the refusals of the Python and
of the C entry points, and the gradient's formula against differences.  Nothing here touches a device."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from drloco_amd import learner_lib as ll
from drloco_amd import lib, memory
from tests import learner_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def L():
    if not os.path.exists(ll.LIB_PATH):
        ll.build()
    return ll.load()


def test_every_declared_symbol_is_exported_and_bound(L):
    text = open(os.path.join(ROOT, 'include', 'drloco_learner.h')).read()
    text = re.sub(r'/\*.*?\*/', '', text, flags=re.S)
    names = sorted(set(re.findall(r'\b(dl_[a-z_0-9]+)\s*\(', text)))
    assert names == sorted(ll._SIGNATURES)
    for n in names:
        assert hasattr(L, n)
    assert L.dl_learner_abi_version() == ll.ABI_VERSION
    assert C.sizeof(ll.MemoryShape) == 11 * 8 + 8
    assert int(re.search(r'#define DL_MEMORY_MARK (\d+)', text).group(1)) == ll.MARK


def test_the_header_is_plain_c(tmp_path):
    import shutil
    import subprocess
    if not shutil.which('gcc'):
        pytest.skip('no gcc')
    for first, second in (('drloco_hip.h', 'drloco_learner.h'), ('drloco_learner.h', 'drloco_learner.h')):
        src = tmp_path / 'a.c'
        src.write_text(f'#include "{first}"\n#include "{second}"\nint main(void) {{ return DL_OK; }}\n')
        subprocess.check_call(['gcc', '-std=c99', '-Wall', '-Werror', '-I' + os.path.join(ROOT, 'include'), '-c', str(src), '-o', str(tmp_path / 'a.o')])


def shape(T=4, N=3, D=8, **kw):
    s = ll.MemoryShape(T=T, N=N, D=D, x_t=N * D, x_n=D, gate_t=N * D, gate_n=D, starts_t=N, starts_n=1, grad_t=N * D, grad_n=D)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


BAD_SHAPES = [dict(dtype=3), dict(dtype=-1), dict(reserved=1), dict(T=-1), dict(N=-1), dict(D=-1), dict(T=1 << 41), dict(T=1 << 30, N=1 << 30), dict(x_t=-1), dict(x_n=-8), dict(gate_t=-1),
              dict(gate_n=-1), dict(starts_t=-1), dict(starts_n=-1), dict(grad_t=-1), dict(grad_n=-1),
              dict(T=(1 << 30) + 1, N=1, D=1), dict(x_n=1 << 28), dict(gate_n=1 << 28), dict(grad_n=1 << 28), dict(T=1, N=1, D=(1 << 29) + 1)]


@pytest.mark.parametrize('bad', BAD_SHAPES, ids=str)
def test_bad_shapes_are_refused_by_every_c_entry(L, bad):
    s = C.byref(shape(**bad))
    p = 4096          # never read: the checks come first
    assert L.dl_memory_workspace_bytes(s) == -1
    assert L.dl_memory_forward(s, p, p, None, None, p, None, None, p, None) == -1
    assert L.dl_memory_backward(s, p, p, None, p, p, None, p, p, None, p, None) == -1
    assert L.dl_memory_step(s, p, p, None, p, p, p, None) == -1
    assert len(L.dl_learner_last_error()) > 5


def test_launches_of_too_many_threads_are_refused(L):
    p = 4096          # never read: the checks come first
    for n in (1 << 33, (1 << 32) + 256, 1 << 40):          # a lane per walker: 2^32 and more of them
        s = C.byref(shape(T=1, N=n, D=1, x_t=0, x_n=1, gate_t=0, gate_n=1, starts_t=0, grad_t=0, grad_n=1))
        assert L.dl_memory_forward(s, p, p, None, None, p, None, None, p, None) == -1
        assert L.dl_memory_backward(s, p, p, None, p, p, None, p, p, None, p, None) == -1
        assert L.dl_memory_step(s, p, p, None, p, p, p, None) == -1
        assert b'too large' in L.dl_learner_last_error()


def test_null_pointers_are_refused(L):
    s, p = C.byref(shape()), 4096
    assert L.dl_memory_workspace_bytes(None) == -1
    for k in (0, 1, 4):
        a = [p, p, None, None, p, None, None, p, None]
        a[k] = None
        assert L.dl_memory_forward(s, *a) == -1
    for k in (0, 1, 3, 6, 7):
        a = [p, p, None, p, p, None, p, p, None, p, None]
        a[k] = None
        assert L.dl_memory_backward(s, *a) == -1
    assert L.dl_memory_forward(s, p, p, None, p, p, p, None, p, None) == -1          # state_out is state
    assert L.dl_memory_backward(s, p, p, None, p, p, p, p, p, p, p, None) == -1      # dstate is grad_state
    assert L.dl_memory_forward(C.byref(shape(T=0)), p, p, None, None, p, None, None, p, None) == -1
    assert L.dl_memory_step(s, p, p, None, p, p, p, None) == -1                      # T is not 1
    one = C.byref(shape(T=1))
    for k in (0, 1, 4, 5):
        a = [p, p, None, p, p, p, None]
        a[k] = None
        assert L.dl_memory_step(one, *a) == -1
    long_ = C.byref(shape(T=100000, N=1, D=64, x_t=64, gate_t=64, grad_t=64))
    assert L.dl_memory_workspace_bytes(long_) > 0
    assert L.dl_memory_forward(long_, p, p, None, None, p, None, None, None, None) == -1          # no workspace
    assert L.dl_memory_backward(long_, p, p, None, p, p, None, p, p, None, None, None) == -1


def test_empty_shapes_are_done_at_once(L):
    for kw in (dict(N=0), dict(D=0)):
        s = C.byref(shape(**kw))
        assert L.dl_memory_workspace_bytes(s) == 0
        assert L.dl_memory_forward(s, None, None, None, None, None, None, None, None, None) == 0
        assert L.dl_memory_backward(s, None, None, None, None, None, None, None, None, None, None, None) == 0
        assert L.dl_memory_step(C.byref(shape(T=1, **kw)), None, None, None, None, None, None, None) == 0


@pytest.mark.parametrize('T,N,D', [(1, 1, 1), (128, 128, 512), (2048, 8, 512), (100003, 1, 333), (65536, 1, 1), (5, 100000, 3), (1 << 20, 2, 64)])
def test_the_workspace_stays_small(L, T, N, D):
    size = L.dl_memory_workspace_bytes(C.byref(shape(T, N, D, x_t=N * D, gate_t=N * D)))
    # a map (two floats) per part of at least 32 steps, and one per eight parts
    assert 0 <= size <= 72 * N * D * (T // 256 + 2) + 64


t3 = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize('args,error', [
    ((t3(4, 3, 8), t3(4, 3, 7)), ValueError),
    ((t3(4, 8), t3(4, 8)), ValueError),
    ((t3(4, 3, 8), t3(4, 3, 8, dtype=torch.bfloat16)), TypeError),
    ((t3(4, 3, 8, dtype=torch.float64), t3(4, 3, 8, dtype=torch.float64)), TypeError),
    ((t3(4, 3, 8), t3(4, 3, 8), t3(4, 3)), TypeError),
    ((t3(4, 3, 8), t3(4, 3, 8), t3(4, 2, dtype=torch.uint8)), ValueError),
    ((t3(4, 3, 8), t3(4, 3, 8), None, t3(3, 7)), ValueError),
    ((t3(4, 3, 8), t3(4, 3, 8), None, t3(3, 8, dtype=torch.bfloat16)), TypeError),
    ((t3(4, 3, 8), [1.0]), TypeError),
    ((t3(4, 3, 8), t3(4, 3, 8)), lib.DrlocoError),          # nothing wrong but the device
])
def test_python_refusals(args, error):
    with pytest.raises(error):
        memory.gated_memory(*args)


@pytest.mark.parametrize('args,kw,error', [
    ((t3(1, 3, 8), t3(1, 3, 8), t3(3, 8)), {}, ValueError),
    ((t3(3, 8), t3(3, 8), None), {}, lib.DrlocoError),
    ((t3(3, 8), t3(3, 8), t3(3, 8, dtype=torch.float16)), {}, TypeError),
    ((t3(3, 8), t3(3, 8), t3(3, 8), t3(4, dtype=torch.uint8)), {}, ValueError),
    ((t3(3, 8), t3(3, 8), t3(3, 8)), {}, lib.DrlocoError),
])
def test_python_refusals_of_a_step(args, kw, error):
    with pytest.raises(error):
        memory.gated_memory_step(*args, **kw)


def test_destinations_of_a_step_are_looked_at():
    x = t3(6, 8)
    for bad in (t3(6, 7), t3(6, 8, dtype=torch.float16), t3(8, 6).t(), x, x[:]):
        with pytest.raises(ValueError):
            memory._destination('out', bad, x, torch.float32, [x])
    both = t3(7, 8)
    with pytest.raises(ValueError):
        memory._destination('out', both[1:], x, torch.float32, [both[:6]])
    assert memory._destination('out', both[1:], x, torch.float32, [both[:1], x]) is not None


def test_the_gradient_formula_against_differences():
    rng = np.random.default_rng(0)
    T, N, D = 9, 3, 2
    x, g, st = rng.standard_normal((T, N, D)), 2 * rng.standard_normal((T, N, D)), rng.standard_normal((N, D))
    starts = rng.random((T, N)) < 0.25
    gh, gl = rng.standard_normal((T, N, D)), rng.standard_normal((N, D))

    def f(x, g, st):
        h, last = R.memory(x, g, starts, st)
        return (h * gh).sum() + (last * gl).sum()
    dx, dg, ds, _ = R.memory_backward(x, g, starts, st, gh, gl)
    e = 1e-6
    for which, grad in ((0, dx), (1, dg), (2, ds)):
        for _ in range(20):
            args = [x.copy(), g.copy(), st.copy()]
            at = tuple(rng.integers(0, n) for n in args[which].shape)
            args[which][at] += e
            up = f(*args)
            args[which][at] -= 2 * e
            # central differences: e^2 of truncation, 2^-53 * |f| / e of rounding
            assert abs((up - f(*args)) / (2 * e) - grad[at]) < 1e-7


@pytest.mark.parametrize('which', [0, 1, 3])
def test_forward_mode_derivatives_are_refused(which):
    """(not dropped: the result would have no tangent, which reads as a zero one)"""
    from torch.autograd import forward_ad
    args = [t3(4, 3, 8), t3(4, 3, 8), None, t3(3, 8)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            memory.gated_memory(*args)
