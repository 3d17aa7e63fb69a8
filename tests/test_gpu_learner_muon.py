"""Orthogonalised updates on the device against their definition in 64 bits (tests/learner_reference.py).

Tolerances, in the Frobenius norm.  With singular values below 1.3 the step p(s) = a s + b s^3 + c s^5 passes an error on at most
4-fold (|p'| <= 4 there).  A step's own error: operands held to 2^-22 twice and lo lo left out, 2^-22 each: below 2^-20; sums of K terms
in 32 bits, signs at random: 2^-24 sqrt(K); each of its three products passes that on by at most a + 2 |b| + 3 |c| = 19 |X|.
bound = sum over steps k of 4^(steps - 1 - k) * 19 * (2^-20 + 2^-24 sqrt(K)) |X_k|.  It is a wide one, so the result is also held against the
same products in float32 (numpy): operands of 22 bits instead of 24 are 4 times as coarse, and left-out terms at most double that:
error <= 8 * (error of float32) + 2^-20 |O|."""
import numpy as np
import pytest
import torch

from tests import learner_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gradient(*shape, seed=0, dtype=torch.float32, scale=1e-3):
    """directions that fall off in strength, and some noise"""
    g = torch.Generator().manual_seed(seed)
    r = min(64, shape[-1], shape[-2])
    fall = torch.arange(1, r + 1, dtype=torch.float32) ** -0.7
    left = torch.randn(*shape[:-1], r, generator=g) * fall
    out = left @ torch.randn(*shape[:-2], r, shape[-1], generator=g) + 0.1 * torch.randn(*shape, generator=g)
    return (out * scale).to(dtype)


def np64(t):
    return t.detach().double().cpu().numpy()


def plain32(g, steps, coefficients):
    a, b, c = (np.float32(v) for v in coefficients)
    x = g.astype(np.float32)
    turned = x.shape[0] > x.shape[1]
    x = x.T if turned else x
    x = (x.astype(np.float64) / max(np.sqrt((x.astype(np.float64) ** 2).sum()), 1e-300)).astype(np.float32)
    for _ in range(steps):
        p = x @ x.T
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.T if turned else x


def check_orthogonal(got, g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), half_step=None):
    """got: [rows, cols] of the device, g: the matrix it was made of, both as tensors"""
    o, g64, trace = np64(got), np64(g), []
    want = R.orthogonal(g64, steps, coefficients, trace)
    norm = np.linalg.norm(want)
    err = np.linalg.norm(o - want)
    k = max(g64.shape)
    bound = sum(4.0 ** (steps - 1 - i) * 19 * (2.0 ** -20 + 2.0 ** -24 * np.sqrt(k)) * x for i, x in enumerate(trace))
    half = (0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2) * norm if half_step is None else half_step
    half += 2.0 ** -25 * np.sqrt(o.size) if got.dtype == torch.float16 else 0.0
    assert err <= bound + half, (err, bound, half)
    err32 = np.linalg.norm(plain32(g64, steps, coefficients) - want)
    assert err <= 8 * err32 + 2.0 ** -20 * norm + half, (err, err32, norm, half)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 7), (7, 1), (1, 512), (8, 512), (512, 8), (29, 512), (512, 29), (16, 16), (31, 33), (32, 32), (64, 64), (65, 63), (33, 129), (127, 128), (130, 257),
                                       (512, 512), (300, 1000), (1000, 300),
                                       (1, 5000), (5000, 1), (15, 1025), (16, 2049), (17, 513), (4000, 30), (32, 1024), (33, 257), (2500, 50), (64, 1000), (63, 9000), (90, 7000), (5000, 130)])
def test_shapes(rows, cols, dtype):
    from drloco_amd.muon import orthogonalise
    g = gradient(rows, cols, seed=rows * 7 + cols, dtype=dtype)
    o = orthogonalise(g.cuda())
    assert o.dtype == dtype and o.shape == g.shape
    check_orthogonal(o, g)


@pytest.mark.parametrize('rows,cols', [(1500, 1700), (1409, 2049), (2300, 1300)])
def test_large_matrices(rows, cols):
    from drloco_amd.muon import orthogonalise
    g = gradient(rows, cols, seed=1)
    check_orthogonal(orthogonalise(g.cuda()), g)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('rows,cols,steps', [(1500, 1700, 5), (1300, 2300, 1), (2050, 1300, 2)])
def test_large_matrices_of_16_bits(rows, cols, steps, dtype):
    """bfloat16: the last step has operands of 11 bits.  Its products are off by 2^-11 / sqrt(3) per operand at random, two operands
    in each of three products: below 2.5 * 2^-11 / sqrt(3) = 2^-10.5 of the norm where singular values differ (2^-9.3 of the norm at most), next to the half step 2^-8
    that check_orthogonal allows.  float16: as exact as float32, one rounding."""
    from drloco_amd.muon import orthogonalise
    g = gradient(rows, cols, seed=2, dtype=dtype)
    check_orthogonal(orthogonalise(g.cuda(), steps), g, steps)


def orthogonal_on_device(g, dtype, steps=5, coefficients=(3.4445, -4.7750, 2.0315)):
    a, b, c = coefficients
    x = g.double()
    x = (x / x.norm()).to(dtype)
    for _ in range(steps):
        p = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
        q = b * p + c * (p @ p)
        x = a * x + (q @ x if x.shape[0] <= x.shape[1] else x @ q)
    return x.double()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('rows,cols', [(2170, 4090), (3904, 4000), (4200, 4096), (700, 20000)])
def test_matrices_that_fill_the_chip(rows, cols, dtype):
    """256 x 128 tiles, whole rounds of them, cut-up rests and a short side that is an odd multiple of 128; 64-bit and float32 products on the
    device, and the second rule of check_orthogonal; bfloat16: next to the half step of the result, 2^-8."""
    from drloco_amd.muon import orthogonalise
    g = gradient(rows, cols, seed=3, dtype=dtype).cuda()
    o, want = orthogonalise(g), orthogonal_on_device(g, torch.float64)
    err, err32, norm = (float(t.norm()) for t in (o.double() - want, orthogonal_on_device(g, torch.float32) - want, want))
    assert err <= 8 * err32 + 2.0 ** -20 * norm + (0 if dtype == torch.float32 else 2.0 ** -8) * norm, (err, err32, norm)


@pytest.mark.parametrize('steps', [1, 2, 3, 8])
@pytest.mark.parametrize('name', ['COEFFICIENTS', 'CUBIC'])
@pytest.mark.parametrize('rows,cols', [(40, 72), (200, 130)])
def test_steps_and_coefficients(rows, cols, steps, name):
    from drloco_amd import muon
    g = gradient(rows, cols, seed=3)
    check_orthogonal(muon.orthogonalise(g.cuda(), steps, getattr(muon, name)), g, steps, getattr(muon, name))


@pytest.mark.parametrize('lead', [(3,), (2, 3), (1,), (17,)])
@pytest.mark.parametrize('rows,cols', [(40, 70), (70, 40), (8, 300), (20, 1100), (1100, 50), (70, 5000)])
def test_batches(lead, rows, cols):
    from drloco_amd.muon import orthogonalise
    g = gradient(*lead, rows, cols, seed=4) * torch.logspace(-3, 3, int(np.prod(lead))).reshape(*lead, 1, 1)
    o = orthogonalise(g.cuda())
    for at in np.ndindex(*lead):
        check_orthogonal(o[at], g[at])
        assert torch.equal(o[at], orthogonalise(g[at].cuda()))


@pytest.mark.parametrize('scale', [1e-38, 1e-30, 1e-10, 1e10, 1e30])
def test_the_size_of_a_gradient_does_not_matter(scale):
    from drloco_amd.muon import orthogonalise
    g = gradient(50, 90, seed=5, scale=1.0) * scale
    assert torch.isfinite(g).all()
    check_orthogonal(orthogonalise(g.cuda()), g)


@pytest.mark.parametrize('rows,cols', [(20, 30), (30, 20), (200, 300), (1, 5), (1500, 20), (100, 5000)])
def test_zeros_stay_zero_and_bad_matrices_keep_to_themselves(rows, cols):
    from drloco_amd.muon import orthogonalise
    g = gradient(5, rows, cols, seed=6).cuda()
    g[1] = 0
    g[2, rows // 2, cols // 3] = float('nan')
    g[3, 0, cols - 1] = float('inf')
    o = orthogonalise(g)
    assert torch.equal(o[1], torch.zeros_like(o[1])) and torch.isnan(o[2]).all() and torch.isnan(o[3]).all()
    assert torch.equal(o[0], orthogonalise(g[0])) and torch.equal(o[4], orthogonalise(g[4]))


def test_matrices_of_one_direction_and_of_equal_ones():
    """rank one: u v' / (|u| |v|) times p^5(1); rows that are orthogonal already: every singular value is 1 / sqrt(m)"""
    from drloco_amd.muon import orthogonalise
    u, v = torch.randn(60, 1, generator=torch.Generator().manual_seed(0)), torch.randn(1, 100, generator=torch.Generator().manual_seed(1))
    check_orthogonal(orthogonalise((u @ v).cuda()), u @ v)
    one = torch.zeros(70, 40)
    one[3, 5] = -2.0
    check_orthogonal(orthogonalise(one.cuda()), one)
    eye = torch.eye(96, 200)
    check_orthogonal(orthogonalise(eye.cuda()), eye)


LAYOUTS = {'transposed': lambda g: g.t().contiguous().cuda().t(), 'wider rows': lambda g: torch.cat((g, g), 1).cuda()[:, :g.shape[1]], 'one element further': lambda g: torch.cat((g[:, :1], g), 1).cuda()[:, 1:],
           'every other row': lambda g: torch.stack((g, g), 1).cuda()[:, 0], 'one row for all': lambda g: g.cuda()}


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16], ids=str)
def test_layouts(layout, dtype):
    from drloco_amd.muon import orthogonalise
    for shape in ((45, 77), (77, 45), (20, 1300), (1300, 40), (130, 200)):
        g = gradient(*shape, seed=7, dtype=dtype)
        placed = LAYOUTS[layout](g)
        want = orthogonalise(g.cuda())
        assert torch.equal(orthogonalise(placed), want)
        row = g[:1].cuda().expand(shape)
        assert torch.equal(orthogonalise(row), orthogonalise(row.contiguous()))
        stack = torch.stack((g, g + g)).cuda().transpose(0, 1)[:, 1]
        assert torch.equal(orthogonalise(stack), orthogonalise(stack.contiguous()))


def test_in_place_and_destinations():
    from drloco_amd.muon import orthogonalise
    for shape in ((45, 77), (300, 200), (2, 9, 30)):
        g = gradient(*shape, seed=8).cuda()
        want = orthogonalise(g)
        out = torch.full_like(g, 7.0)
        assert orthogonalise(g, out=out) is out and torch.equal(out, want)
        version = g._version
        orthogonalise(g, out=g)
        assert torch.equal(g, want) and g._version > version
    with pytest.raises(ValueError):
        orthogonalise(g[0, :, :20].cuda(), out=g[0, :, :20])


@pytest.mark.parametrize('wt', TYPES, ids=str)
@pytest.mark.parametrize('gt', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(29, 40), (512, 29), (130, 200), (29, 1500), (2000, 50)])
def test_the_update(rows, cols, wt, gt):
    from drloco_amd.muon import muon_update
    w, g, m = gradient(rows, cols, seed=1, dtype=wt, scale=0.1), gradient(rows, cols, seed=2, dtype=gt), gradient(rows, cols, seed=3)
    for kw in (dict(lr=0.02, weight_decay=0.01), dict(lr=0.3, beta=0.5, nesterov=False, scale=0.2), dict(lr=0.0), dict(lr=0.1, beta=0.0, steps=3)):
        w2, m2 = muon_update(w.cuda(), g.cuda(), m.cuda(), **kw)
        assert w2.dtype == wt and m2.dtype == torch.float32
        full = dict(beta=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5) | kw
        rw, rm = R.muon(np64(w), np64(g), np64(m), **full)
        # beta, 1 - lr decay and lr scale in 32 bits (2^-24 each), a product and a sum
        assert np.all(np.abs(np64(m2) - rm) <= 3 * 2.0 ** -24 * (np.abs(full['beta'] * np64(m)) + np.abs(np64(g))))
        u = np64(g) + full['beta'] * rm if full['nesterov'] else rm
        gain = full['lr'] * (np.sqrt(max(1.0, rows / cols)) if full['scale'] is None else full['scale'])
        keep = 1 - full['lr'] * full['weight_decay']
        if gain == 0:
            assert torch.equal(w2.cpu(), w)
            continue
        # what was moved, back to an orthogonal factor: u itself is rounded to 32 bits (2^-23 of it, amplified up to 4^steps), weights by half a step of their type
        half = (2.0 ** -22 + (0 if wt == torch.float32 else torch.finfo(wt).eps / 2)) * np.linalg.norm(rw) / gain + 4.0 ** full['steps'] * 2.0 ** -23
        half += 2.0 ** -25 * np.sqrt(w.numel()) / gain if wt == torch.float16 else 0
        check_orthogonal(torch.from_numpy((keep * np64(w) - np64(w2)) / gain).float(), torch.from_numpy(u), full['steps'], half_step=half)


def test_the_update_in_place():
    from drloco_amd.muon import muon_update
    w, g, m = (gradient(2, 45, 77, seed=s).cuda() for s in (1, 2, 3))
    want = muon_update(w, g, m, lr=0.1, weight_decay=0.1)
    w2, m2 = muon_update(w, g, m, lr=0.1, weight_decay=0.1, out=w, momentum_out=m)
    assert w2 is w and m2 is m and torch.equal(w, want[0]) and torch.equal(m, want[1])
    with pytest.raises(ValueError):
        muon_update(w, g, m, lr=0.1, out=m)
    with pytest.raises(ValueError):
        muon_update(w, g, m, lr=0.1, momentum_out=w)
    with pytest.raises(ValueError):
        muon_update(w, g, m, lr=0.1, out=m[:1].expand_as(w))


def test_the_optimiser_and_its_state():
    from drloco_amd.muon import HipMuon
    start = [gradient(64, 29, seed=1, scale=0.1), gradient(64, 64, seed=2, scale=0.1)]
    params = [torch.nn.Parameter(t.cuda()) for t in start]
    opt = HipMuon(params, lr=0.05, weight_decay=0.1)
    ref = [(np64(t), np.zeros(t.shape)) for t in start]
    for k in range(3):
        if k == 2:          # through a checkpoint
            fresh = HipMuon(params, lr=1.0)
            fresh.load_state_dict(opt.state_dict())
            opt = fresh
        for i, p in enumerate(params):
            p.grad = gradient(*p.shape, seed=10 * k + i).cuda()
        before = [p._version for p in params]
        opt.step()
        assert all(p._version > v for p, v in zip(params, before))
        ref = [R.muon(w, np64(p.grad), m, 0.05, weight_decay=0.1) for p, (w, m) in zip(params, ref)]
    for p, (w, m) in zip(params, ref):
        # three steps of 0.05 sqrt(rows / cols) times an orthogonal factor whose error is within the tests above (below 1e-4 of its norm)
        assert np.linalg.norm(np64(p) - w) <= 3 * 0.05 * np.sqrt(max(1, w.shape[0] / w.shape[1])) * 1e-4 * np.sqrt(min(w.shape)) * 1.3
        assert np.abs(np64(opt.state[p]['momentum']) - m).max() <= 9 * 2.0 ** -24 * np.abs(m).max() * 3


def test_the_policy_sees_updated_weights():
    """HipPolicy keeps a packed copy of its weights until their version counter moves"""
    from drloco_amd.muon import HipMuon
    from drloco_amd.policy import HipPolicy
    pol = HipPolicy(hidden=128, seed=0)
    obs = torch.randn(64, 29, device='cuda')
    eps = torch.randn(64, 8, device='cuda')
    pol.forward(obs, eps=eps)
    params = [pol.w1.requires_grad_(), pol.w2.requires_grad_()]
    for p in params:
        p.grad = gradient(*p.shape, seed=3).cuda()
    HipMuon(params, lr=0.1).step()
    with torch.no_grad():
        a, v, lp = pol.forward(obs, eps=eps)
        ra, rv, rlp = pol.torch_reference(obs, eps)
    # float32 products of 29 and 128 terms in another order
    assert (a - ra).abs().max() < 1e-4 and (v - rv).abs().max() < 1e-4


@pytest.mark.parametrize('rows,cols', [(8, 40), (130, 200), (20, 1500), (100, 6000)])
def test_a_captured_update_replays(rows, cols):
    from drloco_amd.muon import muon_update
    w, g, m = (gradient(rows, cols, seed=s).cuda() for s in (1, 2, 3))
    ws, ms = w.clone(), m.clone()
    gs = g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_update(ws, gs, ms, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update(ws, gs, ms, lr=0.1, out=ws, momentum_out=ms)
    for k in range(4):
        gs.copy_(g * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        muon_update(w, g * (k + 1), m, lr=0.1, out=w, momentum_out=m)
        assert torch.equal(w, ws) and torch.equal(m, ms)


def test_two_updates_on_two_streams():
    from drloco_amd.muon import orthogonalise
    g = [gradient(*shape, seed=s).cuda() for s, shape in ((1, (100, 6000)), (2, (110, 7000)))]          # (sums split over workgroups)
    want = [orthogonalise(t) for t in g]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, t in zip(streams, g):
            with torch.cuda.stream(s):
                got.append(orthogonalise(t))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_empty_matrices():
    from drloco_amd.muon import muon_update, orthogonalise
    for shape in ((0, 4), (4, 0), (0, 4, 4)):
        t = torch.zeros(shape, device='cuda')
        assert orthogonalise(t).shape == shape
        assert muon_update(t, t, t, lr=0.1)[0].shape == shape


def test_a_recurrent_policy_learns_through_both():
    """A recurrent policy's update as a learner makes it: layer -> gated memory over the rollout -> action head, gradients through the
    memory, one Muon step of the matrices; against the same in 64 bits on the CPU."""
    from drloco_amd.memory import gated_memory
    from drloco_amd.muon import HipMuon
    T, N, O, D, A = 40, 6, 29, 64, 8
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)
    obs, target, starts = r(T, N, O), r(T, N, A), (torch.rand(T, N, generator=gen) < 0.1).to(torch.uint8)
    ws = [r(D, O) / 5, r(D, O) / 5, r(A, D) / 8]

    def loss_of(x, gate, head, memory, target):
        h = memory(x, gate)
        return ((h @ head.t() - target) ** 2).mean()
    dev = [torch.nn.Parameter(w.cuda()) for w in ws]
    o = obs.cuda()
    loss = loss_of(o @ dev[0].t(), o @ dev[1].t(), dev[2], lambda x, g: gated_memory(x, g, starts.cuda())[0], target.cuda())
    loss.backward()

    def plain(x, gate):
        h, out = torch.zeros(N, D, dtype=torch.float64), []
        a = torch.sigmoid(gate)
        for t in range(T):
            h = torch.where(starts[t].bool()[:, None], 0.0, h)
            h = a[t] * h + (1 - a[t]) * x[t]
            out.append(h)
        return torch.stack(out)
    ref = [w.double().requires_grad_() for w in ws]
    od = obs.double()
    rl = loss_of(od @ ref[0].t(), od @ ref[1].t(), ref[2], plain, target.double())
    rl.backward()
    # float32 throughout: sums of T N = 240 and O = 29 terms, 12 u (T + 1) of the memory: below 1e-4 relative in the norm
    assert abs(float(loss.detach()) - float(rl.detach())) < 1e-4 * float(rl.detach())
    for p, q in zip(dev, ref):
        assert np.linalg.norm(np64(p.grad) - q.grad.numpy()) < 1e-4 * np.linalg.norm(q.grad.numpy())
    grads = [np64(p.grad) for p in dev]
    HipMuon(dev, lr=0.02).step()
    for p, w, g in zip(dev, ws, grads):
        want, _ = R.muon(np64(w), g, np.zeros(g.shape), 0.02)
        scale = 0.02 * np.sqrt(max(1, w.shape[0] / w.shape[1]))
        check_orthogonal((w - p.detach().cpu()) / scale, torch.from_numpy(1.95 * g), half_step=2.0 ** -23 * np.linalg.norm(np64(w)) / scale + 4.0 ** 5 * 2.0 ** -23)
        assert np.linalg.norm(np64(p) - want) < 1e-4 * np.linalg.norm(want)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('batch,rows,cols', [(4, 1024, 2048), (2, 1031, 4099), (7, 900, 1100), (20, 512, 512), (3, 2000, 130), (9, 100, 8000), (16, 833, 833)])
def test_a_matrix_has_the_same_result_in_any_stack(batch, rows, cols, dtype):
    """The tiles' sizes change with the number of matrices (4 x 1024 x 2048 fills the chip with the largest, one does not), the order of an element's sums does not."""
    from drloco_amd.muon import orthogonalise
    g = gradient(batch, rows, cols, seed=8, dtype=dtype).cuda()
    o = orthogonalise(g)
    for k in range(batch):
        assert torch.equal(o[k], orthogonalise(g[k]))


def test_the_training_example_runs_with_muon():
    """Two updates of examples/train_ppo.py: it runs, every weight is finite, the trunk's matrices have moved (nothing is said of the loss)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples', 'train_ppo.py')
    spec = importlib.util.spec_from_file_location('train_ppo', path)
    mod = importlib.util.module_from_spec(spec); spec.loader.exec_module(mod)
    args = dict(n_envs=64, batch=512, minibatch=256, epochs=1, seed=1, log_every=1, quiet=True, return_objects=True, optimizer='muon')
    one, two = (mod.train(mio=mio, **args)[1] for mio in (600e-6, 1100e-6))
    for name in ('w1', 'b1', 'w2', 'b2', 'wa', 'ba', 'wv', 'bv', 'log_std'):
        assert torch.isfinite(getattr(two, name)).all(), name
    for name in ('w1', 'w2', 'wa', 'wv'):
        assert not torch.equal(getattr(one, name), getattr(two, name)), name


@pytest.mark.parametrize('shape', [(8, 512), (3, 20, 1500), (1500, 50), (100, 6000), (600, 130)], ids=str)
def test_everything_in_place(shape):
    from drloco_amd.muon import muon_update, orthogonalise
    w, g, m = (gradient(*shape, seed=s).cuda() for s in (1, 2, 3))
    want, factor = muon_update(w, g, m, lr=0.1, weight_decay=0.1), orthogonalise(g)
    muon_update(w, g, m, lr=0.1, weight_decay=0.1, out=w, momentum_out=m)
    assert torch.equal(w, want[0]) and torch.equal(m, want[1])
    orthogonalise(g, out=g)
    assert torch.equal(g, factor)


def test_a_captured_optimiser_carries_its_momentum():
    from drloco_amd.muon import HipMuon
    shapes = ((64, 29), (20, 1500), (130, 200))
    params, other = ([torch.nn.Parameter(gradient(*s, seed=i, scale=0.1).cuda()) for i, s in enumerate(shapes)] for _ in range(2))
    grads = [gradient(*s, seed=10 + i).cuda() for i, s in enumerate(shapes)]
    opt, eager = HipMuon(params, lr=0.05), HipMuon(other, lr=0.05)
    for p, q, g in zip(params, other, grads):
        p.grad, q.grad = g, g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()          # makes the momenta
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for q, g, i in zip(other, grads, range(3)):
            g.copy_(gradient(*g.shape, seed=20 * k + i))
            q.grad.copy_(g)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for p, q in zip(params, other):
            assert torch.equal(p, q) and torch.equal(opt.state[p]['momentum'], eager.state[q]['momentum'])


@pytest.mark.parametrize('rows,cols', [(8, 512), (3, 700), (2, 40), (16, 1000), (5, 3100), (9, 9000)])
def test_few_rows_are_as_exact_as_32_bits(rows, cols):
    """Over sixteen matrices, so that one lucky rounding says nothing: the mean error is at most that of float32 products.  Of the kernel's roundings
    those of A (22 bits held, some 2^-23 relative) are the larger ones, those of its other products are float32's own; the definition's
    float32 form rounds A's sum too.  A factor of 1.5 for the sampling: errors of single matrices spread by a factor of two, the mean of sixteen by a quarter of it."""
    from drloco_amd.muon import COEFFICIENTS, orthogonalise
    a, b, c = COEFFICIENTS
    g = torch.stack([gradient(rows, cols, seed=100 + k) for k in range(16)])
    got, plain, exact = orthogonalise(g.cuda()).cpu().double(), g.clone(), g.double()
    def steps(x):
        x = x / (x * x).sum(dim=(-2, -1), keepdim=True).sqrt()
        for _ in range(5):
            p = x @ x.transpose(-2, -1).contiguous()
            x = a * x + (b * p + c * (p @ p)) @ x
        return x
    plain, exact = steps(plain).double(), steps(exact)
    off = lambda o: ((o - exact).flatten(1).norm(dim=1) / exact.flatten(1).norm(dim=1)).mean()
    assert off(got) <= 1.5 * off(plain) + 2.0 ** -24


WEIGHTS = {'part of wider rows': lambda w: torch.cat((w, w + 1), -1)[..., :w.shape[-1]], 'transposed': lambda w: w.transpose(-2, -1).contiguous().transpose(-2, -1),
           'every other row': lambda w: torch.stack((w, w + 1), -2).flatten(-3, -2)[..., ::2, :], 'one row for all': lambda w: w[..., :1, :].expand(w.shape)}


@pytest.mark.parametrize('layout', WEIGHTS)
@pytest.mark.parametrize('shape', [(140000, 1), (1, 140000), (131000, 16), (64, 70000), (5000, 1), (900, 1), (2, 140000, 1), (45, 77), (200, 130), (600, 1)], ids=str)
def test_weights_and_momenta_lie_anywhere(shape, layout):
    """Strides of weight, gradient and momentum other than the result's, one column among them on every kernel: the same bits as from contiguous copies."""
    from drloco_amd.muon import muon_update
    w, g, m = (gradient(*shape, seed=s).cuda() for s in (1, 2, 3))
    w, m = WEIGHTS[layout](w), WEIGHTS[layout](m)
    want = muon_update(w.contiguous(), g, m.contiguous(), lr=0.1, weight_decay=0.1)
    got = muon_update(w, WEIGHTS[layout](g) if layout != 'one row for all' else g, m, lr=0.1, weight_decay=0.1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('rows,cols', [(1, 140000), (140000, 1), (16, 131073), (64, 65537), (70000, 33)])
def test_long_sides_beyond_the_slabs(rows, cols, dtype):
    """Short sides of up to 64 whose long side is cut into 256 slabs and more: the kernels of the larger matrices take them."""
    from drloco_amd.muon import orthogonalise
    g = gradient(rows, cols, seed=11, dtype=dtype)
    check_orthogonal(orthogonalise(g.cuda()), g)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('shape', [(8, 512), (512, 29), (20, 1500), (64, 9000), (300, 300), (100, 6000), (700, 900), (1500, 1700), (2050, 1300), (2, 1031, 4099), (4, 1024, 2048), (2170, 4090)], ids=str)
def test_16_bit_results_are_the_32_bit_ones_rounded_once(shape, dtype):
    """The type of a result says how it leaves, not how it is computed: on every kernel it is the float32 result of the same input, rounded to nearest
    (half a step of the type; of float16 half its smallest number too).  A float32 sum that is rounded to float16 at once may differ from
    one that was a float32 number in between by the half step of that, 2^-24."""
    from drloco_amd.muon import muon_update, orthogonalise
    w, g, m = (gradient(*shape, seed=s, dtype=t).cuda() for s, t in ((1, dtype), (2, dtype), (3, torch.float32)))
    w = w / 64          # (small against lr times the factor's entries)
    pairs = [(orthogonalise(g), orthogonalise(g.float())), (orthogonalise(g, 1), orthogonalise(g.float(), 1)),
             (muon_update(w, g, m, lr=0.1, weight_decay=0.1)[0], muon_update(w.float(), g, m, lr=0.1, weight_decay=0.1)[0])]
    for got, full in pairs:
        assert got.dtype == dtype and full.dtype == torch.float32
        if dtype == torch.bfloat16:
            assert torch.equal(got, full.to(dtype))
        else:
            assert bool(((got.double() - full.double()).abs() <= torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -12) * full.double().abs() + 2.0 ** -25).all())


def test_the_training_example_saves_both_optimisers(tmp_path):
    """--optimizer muon --save: Adam's moments of its seven parameters in the zip, the momenta of the trunk's two matrices beside it, both ready to be loaded"""
    import importlib.util
    import io
    import os
    import zipfile
    from drloco_amd import checkpoint
    from drloco_amd.muon import HipMuon
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples', 'train_ppo.py')
    spec = importlib.util.spec_from_file_location('train_ppo', path)
    mod = importlib.util.module_from_spec(spec); spec.loader.exec_module(mod)
    pol = mod.train(mio=1100e-6, n_envs=64, batch=512, minibatch=256, epochs=1, seed=1, log_every=1, quiet=True, return_objects=True, optimizer='muon', save_path=str(tmp_path))[1]
    names = sorted(os.listdir(tmp_path / 'models'))
    assert [n.split('_')[0] for n in names] == ['model', 'muon']
    with zipfile.ZipFile(tmp_path / 'models' / names[0]) as z:
        adam = torch.load(io.BytesIO(z.read('policy.optimizer.pth')), weights_only=True)
    order = list(checkpoint._PARAM_ORDER)
    assert sorted(order[i] for i in adam['state']) == sorted(set(order) - {'w1', 'w2'})
    assert all(bool(torch.isfinite(s['exp_avg']).all()) and float(s['step']) > 0 for s in adam['state'].values())
    params = [torch.nn.Parameter(getattr(pol, n).detach().clone()) for n in ('w1', 'w2')]
    opt = HipMuon(params)
    opt.load_state_dict(torch.load(tmp_path / 'models' / names[1], weights_only=True))
    for p in params:
        m = opt.state[p]['momentum']
        assert m.shape == p.shape and m.dtype == torch.float32 and float(m.abs().sum()) > 0


def test_what_the_library_refuses_is_a_drloco_error():
    """as everywhere in the package: here more matrices than a launch takes"""
    from drloco_amd import lib
    from drloco_amd.muon import muon_update, orthogonalise
    many = torch.zeros(1, 2, 2, device='cuda').expand(65536, 2, 2)
    with pytest.raises(lib.DrlocoError, match='65535'):
        orthogonalise(many)
    with pytest.raises(lib.DrlocoError, match='65535'):
        muon_update(many, many, many, lr=0.1)
