"""The gated memory on the device against its definition in 64 bits (tests/learner_reference.py).

Tolerances.  u = 2^-24.  One step rounds at most: the gate's small side (4 u relative: exponential, sum, reciprocal, product), the
difference, the product-sum; with |x|, |h| <= M each step adds at most 8 u M to h, and h's error passes on by a factor a <= 1, so
after T steps |error| <= 8 u M T (joining the maps of runs multiplies rounded products of a: at most 4 u per step again, 4 u M T).
State: 12 u M (T + 1).  h is rounded once more, half a step of its type: eps / 2 * |h|.  A gradient l that reaches a step obeys the
same recurrence: 12 u L (T + 1) with L = max |l|; dx multiplies by s (4 u more); dgate multiplies l a s <= L / 4 with h - x <= 2 M:
(error of h) L / 4 + 2 M / 4 (error of l) + 16 u M L.  A 16-bit type adds its half step, and half its smallest subnormal."""
import numpy as np
import pytest
import torch

from tests import learner_reference as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def rounding(t, value):
    return (0 if t == torch.float32 else torch.finfo(t).eps / 2) * np.abs(value) + TINY[t]


def make(T, N, D, dtype, starts='some', state=True, seed=0, spread=2.0, shift=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, N, D, generator=g).to(dtype)
    gate = (torch.randn(T, N, D, generator=g) * spread + shift).to(dtype)
    st = torch.randn(N, D, generator=g) if state else None
    b = {'none': None, 'some': (torch.rand(T, N, generator=g) < 0.1).to(torch.uint8), 'all': torch.ones(T, N, dtype=torch.uint8), 'first': torch.zeros(T, N, dtype=torch.uint8)}[starts]
    if starts == 'first':
        b[0] = 7
    gh, gl = torch.randn(T, N, D, generator=g).to(dtype), torch.randn(N, D, generator=g)
    return x, gate, b, st, gh, gl


def np64(t):
    return None if t is None else t.double().numpy()


def dev(t):
    return None if t is None else t.cuda()


def check_all(x, gate, b, st, gh, gl, place=dev, state_grad=True):
    """Forward and backward of the device against 64 bits; `place` puts a [T, N, D] input on the device in some layout."""
    from drloco_amd.memory import gated_memory
    T, dt = x.shape[0], x.dtype
    xd, gd, sd = place(x).requires_grad_(), place(gate).requires_grad_(), dev(st)
    if sd is not None and state_grad:
        sd.requires_grad_()
    h, last = gated_memory(xd, gd, dev(b), sd)
    assert h.dtype == dt and last.dtype == torch.float32 and h.shape == x.shape
    h_, last_ = R.memory(np64(x), np64(gate), b, np64(st))
    M = max(np.abs(np64(x)).max(), 0 if st is None else np.abs(np64(st)).max())
    eh = 12 * U * M * (T + 1)
    assert np.all(np.abs(np64(last.detach().cpu()) - last_) <= eh)
    assert np.all(np.abs(np64(h.detach().cpu()) - h_) <= eh + rounding(dt, h_))
    leaves = [xd, gd] + ([sd] if sd is not None and state_grad else [])
    outs, grads = ([h], [place(gh)]) if gl is None else ([last], [dev(gl)]) if gh is None else ([h, last], [place(gh), dev(gl)])
    got = torch.autograd.grad(outs, leaves, grads)
    dx, dg, ds, L = R.memory_backward(np64(x), np64(gate), b, np64(st), np64(gh), np64(gl))
    el = 12 * U * L * (T + 1)
    assert np.all(np.abs(np64(got[0].cpu()) - dx) <= el + 4 * U * L + rounding(dt, dx))
    assert np.all(np.abs(np64(got[1].cpu()) - dg) <= eh * L / 4 + el * M / 2 + 16 * U * M * L + rounding(dt, dg))
    if len(got) > 2:
        assert np.all(np.abs(np64(got[2].cpu()) - ds) <= el)
    return h, last, got


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('T', [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 300])
@pytest.mark.parametrize('N,D', [(1, 1), (3, 5), (2, 6), (7, 36), (1, 64), (5, 130)])
def test_rollouts(T, N, D, dtype):
    check_all(*make(T, N, D, dtype, seed=T * 1000 + D))


@pytest.mark.parametrize('starts', ['none', 'some', 'all', 'first'])
@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('which', ['h', 'last', 'both'])
def test_starts_states_and_missing_gradients(starts, state, which):
    x, gate, b, st, gh, gl = make(37, 6, 20, torch.float32, starts, state, seed=3)
    check_all(x, gate, b, st, None if which == 'last' else gh, None if which == 'h' else gl)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('T,N,D', [(2049, 1, 3), (2048, 2, 64), (1111, 3, 7), (5000, 1, 128)])
def test_long_rollouts_of_few_walkers(T, N, D, dtype):
    """few columns: the time axis is cut over workgroups"""
    x, gate, b, st, gh, gl = make(T, N, D, dtype, seed=T)
    b = (torch.rand(T, N, generator=torch.Generator().manual_seed(1)) < 0.002).to(torch.uint8)
    check_all(x, gate, b, st, gh, gl)
    check_all(x, gate, None, st, gh, gl)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('T', [8191, 8192, 8193, 8320, 8321, 16385, 25000])
def test_chains_of_several_groups(T, dtype):
    """64 workgroups of 128 steps each hand a value to the next 64: rollouts around and over multiples of 8192 steps, episodes that
    begin right there, and none at all"""
    x, gate, _, st, gh, gl = make(T, 2, 5, dtype, seed=T, shift=4.0)
    b = torch.zeros(T, 2, dtype=torch.uint8)
    b[[0, 127, 128, 8190, T - 1], 0] = 1
    if T > 8192:
        b[8192, 1] = 1
    check_all(x, gate, b, st, gh, gl)
    check_all(x, gate, None, st, gh, gl)


@pytest.mark.parametrize('T,N,D', [(20, 513, 256), (40, 2100, 66), (129, 300, 512)])
def test_many_walkers(T, N, D):
    check_all(*make(T, N, D, torch.bfloat16, seed=5))


LAYOUTS = {
    'walker-major': lambda t: t.transpose(0, 1).contiguous().cuda().transpose(0, 1),
    'part of wider rows': lambda t: torch.cat((t, t), 2).cuda()[..., :t.shape[2]],
    'one element further': lambda t: torch.cat((t[..., :1], t), 2).cuda()[..., 1:],
    'every other step': lambda t: torch.stack((t, t), 1).cuda()[:, 0],
    'last axis apart': lambda t: t.transpose(1, 2).contiguous().cuda().transpose(1, 2),
}


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
def test_layouts(layout, dtype):
    def place(t):
        out = LAYOUTS[layout](t).detach()
        assert torch.equal(out.cpu(), t)
        return out
    check_all(*make(50, 6, 24, dtype, seed=9), place=place)


def test_broadcast_inputs_and_their_gradients():
    """x shared by all walkers, gates shared by all steps: strides of 0, gradients summed by autograd"""
    from drloco_amd.memory import gated_memory
    x, gate, b, st, gh, gl = make(33, 5, 16, torch.float32, seed=2)
    x1, g1, s1 = x[:, :1].cuda().requires_grad_(), gate[:1].cuda().requires_grad_(), st[:1].cuda().requires_grad_()
    h, last = gated_memory(x1.expand(33, 5, 16), g1.expand(33, 5, 16), b.cuda(), s1.expand(5, 16))
    xf, gf, sf = x[:, :1].expand_as(x), gate[:1].expand_as(gate), st[:1].expand_as(st)
    h_, last_ = R.memory(np64(xf), np64(gf), b, np64(sf))
    M = float(max(x.abs().max(), st.abs().max()))
    eh = 12 * U * M * 34
    assert np.all(np.abs(np64(h.detach().cpu()) - h_) <= eh)
    # (a gradient that is broadcast itself: all its strides are 0)
    got = torch.autograd.grad(h.sum(), [x1, g1, s1])
    dx, dg, ds, L = R.memory_backward(np64(xf), np64(gf), b, np64(sf), np.ones((33, 5, 16)), None)
    el = 12 * U * L * 34
    # sums of 5, 33 and 5 terms: their errors add up, and each addition rounds once more
    assert np.all(np.abs(np64(got[0].cpu())[:, 0] - dx.sum(1)) <= 5 * (el + 4 * U * L) + 5 * U * np.abs(dx).sum(1))
    assert np.all(np.abs(np64(got[1].cpu())[0] - dg.sum(0)) <= 33 * (eh * L / 4 + el * M / 2 + 16 * U * M * L) + 33 * U * np.abs(dg).sum(0))
    assert np.all(np.abs(np64(got[2].cpu())[0] - ds.sum(0)) <= 5 * el + 5 * U * np.abs(ds).sum(0))


@pytest.mark.parametrize('T,N,D', [(64, 4, 32), (3000, 1, 8)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_nothing_leaks_over_the_start_of_an_episode(T, N, D, bad):
    """NaN and infinities before a start: neither the memory behind it nor the gradients of the steps behind it see them, and
    a NaN in a gradient behind it does not reach the steps before."""
    from drloco_amd.memory import gated_memory
    x, gate, _, st, gh, gl = make(T, N, D, torch.float32, 'none', seed=4)
    cut = T // 2 + 5
    b = torch.zeros(T, N, dtype=torch.uint8)
    b[cut] = 1
    x2, st2, gate2 = x.clone(), st.clone(), gate.clone()
    x2[cut - 3] = bad
    st2[:] = bad
    gate2[cut - 7] = float('nan')
    leaves = [t.cuda().requires_grad_() for t in (x2, gate2, st2)]
    h, last = gated_memory(leaves[0], leaves[1], b.cuda(), leaves[2])
    clean = [t.cuda().requires_grad_() for t in (x, gate, st)]
    hc, lastc = gated_memory(clean[0], clean[1], b.cuda(), clean[2])
    assert torch.equal(h[cut:], hc[cut:]) and torch.equal(last, lastc) and torch.isfinite(last).all()
    assert not torch.isfinite(h[cut - 3]).any()
    a = torch.autograd.grad([h, last], leaves, [gh.cuda(), gl.cuda()], retain_graph=True)
    c = torch.autograd.grad([hc, lastc], clean, [gh.cuda(), gl.cuda()], retain_graph=True)
    for p, q in zip(a[:2], c[:2]):
        assert torch.equal(p[cut:], q[cut:]) and torch.isfinite(p[cut:]).all()
    gh2 = gh.clone()
    gh2[cut:] = bad
    d = torch.autograd.grad([hc], clean, [gh2.cuda()])
    e = torch.autograd.grad([gated_memory(*[t for t in clean[:2]], b.cuda(), clean[2])[0]], clean, [torch.cat((gh[:cut], torch.zeros_like(gh[cut:]))).cuda()])
    for p, q in zip(d[:2], e[:2]):
        assert torch.equal(p[:cut], q[:cut])
    assert torch.equal(d[2], e[2])


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_closed_and_open_gates_are_exact(dtype):
    """gates of the type's largest and lowest values and infinite ones: h is x, or the state as it was"""
    from drloco_amd.memory import gated_memory
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn(40, 3, 8, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    st = torch.randn(3, 8, generator=torch.Generator().manual_seed(1)).cuda()
    for low in (lo, -float('inf')):
        h, last = gated_memory(x, torch.full_like(x, low), None, 1e6 * st)
        assert torch.equal(h, x) and torch.equal(last, x[-1].float())
    for high in (hi, float('inf')):
        h, last = gated_memory(x, torch.full_like(x, high), None, st)
        assert torch.equal(last, st) and torch.equal(h, st.to(dtype).expand_as(h))


def test_a_long_memory_keeps_its_precision():
    """gate = 10: 45 thousandths of a percent are taken in per step.  With a rounded to 32 bits the sums would be off by 2^-25 / (1 - a)
    = 6.6e-4 relative; the form used here rounds h once a step, at random: 30 000 steps, and the bound counts every one as half a unit."""
    from drloco_amd.memory import gated_memory
    T = 30000
    x = (1 + torch.rand(T, 1, 4, generator=torch.Generator().manual_seed(0))).cuda()
    gate = torch.full_like(x, 10.0)
    h, last = gated_memory(x, gate)
    h_, last_ = R.memory(np64(x.cpu()), np64(gate.cpu()))
    # rounding of h: at most u * 2 a step, kept for 1 / (1 - a) = 22027 steps; measured far below because its signs differ
    assert np.all(np.abs(np64(last.cpu()) - last_) <= 2 * U * 22027 * 2)
    assert np.abs(np64(last.cpu()) - last_).max() / last_.min() < 6.6e-4 / 20


def test_offsets_beyond_32_bits():
    """more than 2^31 elements: the last walkers' channels and the last steps are right"""
    from drloco_amd.memory import gated_memory
    T, N, D = 2100, 1025, 1024
    x = torch.zeros(T, N, D, dtype=torch.bfloat16, device='cuda')
    gate = torch.zeros(T, N, D, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator().manual_seed(0)
    cols = [0, 511, 1024]
    xs, gs = torch.randn(T, 3, D, generator=g).to(torch.bfloat16), torch.randn(T, 3, D, generator=g).to(torch.bfloat16)
    x[:, cols], gate[:, cols] = xs.cuda(), gs.cuda()
    x.requires_grad_(), gate.requires_grad_()
    h, last = gated_memory(x, gate)
    h_, last_ = R.memory(np64(xs), np64(gs))
    M = float(xs.abs().max())
    assert np.all(np.abs(np64(last[cols].detach().cpu()) - last_) <= 12 * U * M * (T + 1))
    assert np.all(np.abs(np64(h[:, cols].detach().cpu()) - h_) <= 12 * U * M * (T + 1) + rounding(torch.bfloat16, h_))
    assert float(h[:, 1].detach().abs().max()) == 0.0
    grad = torch.zeros_like(h)
    ghs = torch.randn(T, 3, D, generator=g).to(torch.bfloat16)
    grad[:, cols] = ghs.cuda()
    dx, dg = torch.autograd.grad(h, [x, gate], grad)
    del grad, h
    rx, rg, _, L = R.memory_backward(np64(xs), np64(gs), None, None, np64(ghs), None)
    el, eh = 12 * U * L * (T + 1), 12 * U * M * (T + 1)
    assert np.all(np.abs(np64(dx[:, cols].cpu()) - rx) <= el + 4 * U * L + rounding(torch.bfloat16, rx))
    assert np.all(np.abs(np64(dg[:, cols].cpu()) - rg) <= eh * L / 4 + el * M / 2 + 16 * U * M * L + rounding(torch.bfloat16, rg))


def test_walkers_far_apart():
    """walker-major with more than 2^29 elements under the lanes of a wave: the wrapper makes a time-major copy"""
    far = 1 << 23
    store = torch.zeros(69 * far + 64, dtype=torch.float16, device='cuda')
    place = lambda t: store.as_strided(t.shape, (t.shape[2], far, 1)).copy_(t).detach()
    x, gate, b, st, gh, gl = make(5, 70, 4, torch.float16, seed=3)
    check_all(x, gate, b, st, gh, gl, place=lambda t: place(t).clone(memory_format=torch.preserve_format) if t is gh else place(t) if t is x else t.cuda())


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,D', [(1, 1), (8, 512), (3, 7), (65, 30), (4096, 64)])
def test_steps_are_the_rollout_bit_for_bit(N, D, dtype):
    from drloco_amd.memory import gated_memory, gated_memory_step
    T = 12          # within one run of the rollout kernel: the same operations in the same order
    x, gate, b, st, _, _ = (dev(t) for t in make(T, N, D, dtype, seed=N))
    h, last = gated_memory(x, gate, b, st)
    state = st.clone()
    out = torch.empty_like(h)
    for t in range(T):
        o, s2 = gated_memory_step(x[t], gate[t], state, b[t].bool() if t % 2 else b[t], out=out[t], state_out=state)
        assert s2.data_ptr() == state.data_ptr() and o.data_ptr() == out[t].data_ptr()
    assert torch.equal(out, h) and torch.equal(state, last)
    o, fresh = gated_memory_step(x[0], gate[0], st)
    h0, _ = gated_memory(x[:1], gate[:1], None, st)
    assert torch.equal(o, h0[0]) and fresh.data_ptr() != st.data_ptr()


def test_a_step_in_other_layouts():
    from drloco_amd.memory import gated_memory, gated_memory_step
    x, gate, b, st, _, _ = (dev(t) for t in make(1, 9, 20, torch.float32, seed=1))
    want, wl = gated_memory(x, gate, b, st)
    for f in (lambda t: torch.cat((t[..., :1], t), -1)[..., 1:], lambda t: t.t().contiguous().t(), lambda t: torch.stack((t, t), 1)[:, 0]):
        o, s = gated_memory_step(f(x[0]), f(gate[0]), f(st), torch.stack((b[0], b[0]), 1)[:, 0])
        assert torch.equal(o, want[0]) and torch.equal(s, wl)
    o, s = gated_memory_step(x[0, :1].expand(9, 20), gate[0], st)
    w2, s2 = gated_memory(x[:, :1].expand(1, 9, 20), gate, None, st)
    assert torch.equal(o, w2[0]) and torch.equal(s, s2)


def test_empty_calls():
    from drloco_amd.memory import gated_memory, gated_memory_step
    st = torch.randn(3, 4, device='cuda', requires_grad=True)
    x = torch.zeros(0, 3, 4, device='cuda', requires_grad=True)
    h, last = gated_memory(x, x, None, st)
    assert h.shape == (0, 3, 4) and torch.equal(last, st)
    last.sum().backward()
    assert torch.equal(st.grad, torch.ones_like(st))
    for shape in ((5, 0, 4), (5, 3, 0)):
        h, last = gated_memory(torch.zeros(shape, device='cuda'), torch.zeros(shape, device='cuda'))
        assert h.shape == shape and last.shape == shape[1:]
    o, s = gated_memory_step(torch.zeros(0, 4, device='cuda'), torch.zeros(0, 4, device='cuda'), torch.zeros(0, 4, device='cuda'))
    assert o.shape == s.shape == (0, 4)


def test_refusals_on_the_device():
    from drloco_amd import lib
    from drloco_amd.memory import gated_memory, gated_memory_step
    x = torch.zeros(4, 3, 8, device='cuda')
    with pytest.raises(lib.DrlocoError):
        gated_memory(x, x, torch.zeros(4, 3, dtype=torch.uint8))
    with pytest.raises(ValueError):
        gated_memory_step(x[0], x[0], torch.zeros(3, 8, device='cuda'), out=torch.zeros(3, 8, device='cuda', dtype=torch.float16))
    both = torch.zeros(4, 8, device='cuda')
    with pytest.raises(ValueError):
        gated_memory_step(x[0], x[0], both[:3], state_out=both[1:])
    with pytest.raises(ValueError):
        gated_memory_step(x[0], x[1], both[:3], out=x[0])
    xr = x.clone().requires_grad_()
    h, _ = gated_memory(xr, x)
    gx, = torch.autograd.grad(h.sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.parametrize('T,N,D', [(40, 16, 64), (3000, 1, 64)])
def test_a_captured_pass_replays(T, N, D):
    """forward and backward in a HIP graph, replayed over changed inputs between eager calls"""
    from drloco_amd.memory import gated_memory
    x, gate, b, st, gh, gl = (dev(t) for t in make(T, N, D, torch.float32, seed=6))
    xs, gs, ss = (t.clone().requires_grad_() for t in (x, gate, st))

    def passes(p, q, r):
        h, last = gated_memory(p, q, b, r)
        return (h, last) + torch.autograd.grad([h, last], [p, q, r], [gh, gl])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(xs, gs, ss)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = passes(xs, gs, ss)
    for k in range(4):
        with torch.no_grad():
            xs.copy_(x * (k + 1)), gs.copy_(gate - k), ss.copy_(st + k)
        graph.replay()
        torch.cuda.synchronize()
        want = passes(xs.detach().clone().requires_grad_(), gs.detach().clone().requires_grad_(), ss.detach().clone().requires_grad_())
        for p, q in zip(outs, want):
            assert torch.equal(p, q)


def test_two_calls_on_two_streams():
    from drloco_amd.memory import gated_memory
    data = [[dev(t) for t in make(4000, 1, 96, torch.float32, seed=s)] for s in (1, 2)]
    want = [gated_memory(*d[:4]) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(gated_memory(*d[:4]))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1])


def test_the_same_tensor_for_x_and_gate():
    from drloco_amd.memory import gated_memory
    x = torch.randn(20, 3, 8, device='cuda', requires_grad=True)
    h, _ = gated_memory(x, x)
    g, = torch.autograd.grad(h.sum(), x)
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    h2, _ = gated_memory(a, b)
    ga, gb = torch.autograd.grad(h2.sum(), [a, b])
    assert torch.equal(h, h2) and torch.equal(g, ga + gb)


def test_repeats_are_bit_identical():
    x, gate, b, st, gh, gl = make(2500, 2, 40, torch.bfloat16, seed=8)
    first = check_all(x, gate, b, st, gh, gl)
    second = check_all(x, gate, b, st, gh, gl)
    assert torch.equal(first[0], second[0]) and all(torch.equal(p, q) for p, q in zip(first[2], second[2]))


@pytest.mark.parametrize('which', [0, 1, 3])
def test_forward_mode_derivatives_are_refused(which):
    from torch.autograd import forward_ad
    from drloco_amd.memory import gated_memory
    x, gate, b, st, _, _ = (dev(t) for t in make(9, 3, 8, torch.float32))
    args = [x, gate, b, st]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for grad in (False, True):
            x.requires_grad_(grad)
            with pytest.raises(RuntimeError):
                gated_memory(*args)
        args[which] = forward_ad.unpack_dual(args[which]).primal.detach()
        gated_memory(*args)


def test_transforms_are_refused_or_right():
    """torch.func's wrapped tensors have no memory for a kernel to read: an error, not a wrong result"""
    from drloco_amd.memory import gated_memory
    x, gate, b, st, _, _ = (dev(t) for t in make(9, 3, 8, torch.float32))
    f = lambda v: gated_memory(v, gate, b, st)[0].sum()
    for call in (lambda: torch.func.grad(f)(x), lambda: torch.vmap(f)(torch.stack((x, x))), lambda: torch.func.jvp(f, (x,), (x,))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize('T', [1, 7, 16, 17, 100, 128, 129, 300, 2050, 9000])
@pytest.mark.parametrize('N,D', [(1, 5), (3, 64), (600, 130)])
def test_the_state_is_the_last_step(T, N, D):
    """state = h[T-1] before it is rounded: the same bits in float32, also where the last step takes in an infinity, whatever the form"""
    from drloco_amd.memory import gated_memory
    if T * N * D > 3e7:
        T = 300
    x, gate, b, st, _, _ = (dev(t) for t in make(T, N, D, torch.float32, seed=T))
    h, last = gated_memory(x, gate, b, st)
    assert torch.equal(h[-1], last)
    bad = x.clone()
    bad[-1, :, 0], bad[-1, :, 1], bad[-1, :, 2] = float('inf'), -float('inf'), float('nan')
    h2, last2 = gated_memory(bad, gate, b, st)
    assert torch.equal(h2[-1].nan_to_num(1.5, 2.5, 3.5), last2.nan_to_num(1.5, 2.5, 3.5)) and not torch.isfinite(last2[:, :3]).any()
    assert torch.equal(last2[:, 3:], last[:, 3:]) and torch.equal(h2[:-1], h[:-1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('T,N,D', [(1, 3, 5), (12, 5, 8), (128, 2, 7), (300, 3, 20), (2000, 2, 6), (9000, 1, 5), (40, 2100, 66)])
def test_the_largest_numbers(T, N, D, dtype):
    """x and state of up to the type's largest number, of either sign and next to small ones: every h lies between them, so nothing may
    be infinite, though x - h is beyond float32 and joined states are rounded against its end"""
    x, gate, b, st, gh, gl = make(T, N, D, dtype, seed=T)
    g = torch.Generator().manual_seed(T)
    most = torch.finfo(dtype).max
    big = lambda *s: (torch.randint(0, 2, s, generator=g) * 2 - 1).float() * most
    x = torch.where(torch.rand(T, N, D, generator=g) < 0.7, big(T, N, D), x.float()).to(dtype)
    st = torch.where(torch.rand(N, D, generator=g) < 0.7, big(N, D), st)
    x[:, :, 1], st[:, 1] = most, most          # a channel that stays there
    h, last, got = check_all(x, gate, b, st, gh * 2.0 ** -10, gl * 2.0 ** -10)
    assert torch.isfinite(h).all() and torch.isfinite(last).all() and all(torch.isfinite(t).all() for t in got)
    if T == 1:
        from drloco_amd.memory import gated_memory_step
        o, s = gated_memory_step(x[0].cuda(), gate[0].cuda(), st.cuda(), b[0].cuda())
        assert torch.equal(o, h[0]) and torch.equal(s, last)


@pytest.mark.parametrize('T,N,D', [(1, 3, 5), (128, 2, 7), (2000, 2, 6), (40, 2100, 66)])
def test_the_largest_state_of_a_float16_memory(T, N, D):
    from drloco_amd.memory import gated_memory
    x, gate, _, st, _, _ = make(T, N, D, torch.float16, seed=T, shift=6.0)
    most = torch.finfo(torch.float32).max
    x, st = torch.sign(x) * torch.finfo(torch.float16).max, torch.sign(st) * most
    gate[:, :, 1] = float('inf')          # a channel that stays there
    _, last = gated_memory(x.cuda(), gate.cuda(), None, st.cuda())
    _, last_ = R.memory(np64(x), np64(gate), None, np64(st))
    assert torch.isfinite(last).all() and np.all(np.abs(np64(last.cpu()) - last_) <= 12 * U * most * (T + 1)) and torch.equal(last[:, 1].cpu(), st[:, 1])


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_a_captured_step_replays(dtype):
    """a control step in a graph, the state kept in place, replayed over new inputs with eager steps between"""
    from drloco_amd.memory import gated_memory_step
    x, gate, b, st, _, _ = (dev(t) for t in make(6, 7, 20, dtype, seed=2))
    xs, gs, bs, state, eager, out = x[0].clone(), gate[0].clone(), b[0].clone(), st.clone(), st.clone(), torch.empty_like(x[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_memory_step(xs, gs, st, bs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gated_memory_step(xs, gs, state, bs, out=out, state_out=state)
    for t in range(6):
        xs.copy_(x[t]), gs.copy_(gate[t]), bs.copy_(b[t])
        graph.replay()
        h, _ = gated_memory_step(x[t], gate[t], eager, b[t], state_out=eager)
        torch.cuda.synchronize()
        assert torch.equal(out, h) and torch.equal(state, eager)
