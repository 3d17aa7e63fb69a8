"""The learner's operators as a user's program calls them, for measurement: the gated memory of a recurrent policy (one control
step, a whole rollout, a whole rollout with its gradients), the orthogonalisation of an update and the weight update built on it.

With `own` false, `run` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end); with
`own` true it calls drloco_amd.memory and drloco_amd.muon."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def listed():
    return [
        # the reference's eight walkers, one control step: what a policy in the loop waits for
        dict(name='step_eight', op='step', T=1, N=8, D=512, type='f32', every=300, state=True),
        # one control step of a whole fleet on one GPU
        dict(name='step_fleet', op='step', T=1, N=4096, D=512, type='bf16', every=300, state=True),
        # twenty evaluation episodes at the episode limit, replayed through the memory (no gradients)
        dict(name='scan_evaluation', op='scan', T=3000, N=20, D=256, type='f32', every=0, state=True),
        # one walker's long log of episodes in an odd width: few rows, the work lies along the time axis
        dict(name='scan_log', op='scan', T=100003, N=1, D=333, type='f16', every=1500, state=False),
        # the reference's rollout, 8 walkers x 2048 steps, with gradients
        dict(name='train_reference', op='train', T=2048, N=8, D=512, type='f32', every=300, state=True),
        # the training example's rollout, 128 walkers x 128 steps
        dict(name='train_rollout', op='train', T=128, N=128, D=512, type='bf16', every=100, state=True),
        # the benchmark's rollout, 4096 walkers x 512 steps
        dict(name='train_fleet', op='train', T=512, N=4096, D=128, type='bf16', every=300, state=True),
        # the gradient of the action head
        dict(name='orth_head', op='orth', B=1, m=8, n=512, type='f32'),
        # the gradient of the trunk's square layer
        dict(name='orth_trunk', op='orth', B=1, m=512, n=512, type='f32'),
        # a large generic layer
        dict(name='orth_large', op='orth', B=1, m=4096, n=8192, type='bf16'),
        # the first layer of the policy: tall, odd width
        dict(name='muon_first', op='muon', B=1, m=512, n=29, type='f32'),
        # two stacked odd-sized layers with 16-bit weights
        dict(name='muon_stack', op='muon', B=2, m=1031, n=4099, type='bf16'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['step', 'scan', 'train', 'orth', 'muon'])
    kind = rng.choice(['f32', 'bf16', 'f16'])
    if op in ('orth', 'muon'):
        m, n = _log(rng, 1, 4096), _log(rng, 1, 8000)
        return dict(op=op, B=_log(rng, 1, 4) if m * n < 4000000 else 1, m=m, n=n, type=kind)
    D = _log(rng, 1, 1024)
    if op == 'step':
        return dict(op=op, T=1, N=_log(rng, 1, 8192), D=D, type=kind, every=rng.choice([0, 20, 300]), state=True)
    T = _log(rng, 2, 100000)
    N = _log(rng, 1, max(1, min(4096, 100000000 // (T * D))))
    return dict(op=op, T=T, N=N, D=D, type=kind, every=rng.choice([0, 20, 300, 3000]), state=rng.random() < 0.7)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    dt = TYPES[case['type']]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device='cuda') * scale + shift).to(dtype)

    s = {'case': case}
    if case['op'] in ('orth', 'muon'):
        B, m, n = case['B'], case['m'], case['n']
        # a minibatch gradient: a sum of outer products whose directions fall off in strength, and some noise
        r = min(256, m, n)
        fall = torch.arange(1, r + 1, device='cuda', dtype=torch.float32) ** -0.7
        g = torch.bmm(torch.randn(B, m, r, generator=gen, device='cuda') * fall, torch.randn(B, r, n, generator=gen, device='cuda'))
        g = (g + 0.1 * torch.randn(B, m, n, generator=gen, device='cuda')) * 1e-3
        s['g'] = g.to(dt)
        if case['op'] == 'muon':
            s['w'] = normal(B, m, n, scale=1.0 / math.sqrt(n))
            s['m'] = g * 4.0 + normal(B, m, n, scale=1e-3, dtype=torch.float32)
        if B == 1:
            s.update({k: v[0] for k, v in s.items() if k in ('g', 'w', 'm')})
        return s
    T, N, D = case['T'], case['N'], case['D']
    shape = (N, D) if case['op'] == 'step' else (T, N, D)
    train = case['op'] == 'train'
    s['x'] = normal(*shape).requires_grad_(train)
    # forget gates from a few steps to a few hundred, as a bias per channel plus what the input says
    s['gate'] = (normal(*shape, dtype=torch.float32) + normal(D, scale=1.5, shift=2.0, dtype=torch.float32)).to(dt).requires_grad_(train)
    every = case['every']
    s['starts'] = (torch.rand(*shape[:-1], generator=gen, device='cuda') * every < 1).to(torch.uint8) if every else None
    s['state'] = normal(N, D, dtype=torch.float32).requires_grad_(train) if case['state'] else None
    if train:
        s['grad'] = normal(T, N, D, scale=1e-2)
        s['grad_state'] = normal(N, D, scale=1e-2, dtype=torch.float32)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _scan(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along the first axis: each pass joins runs of k steps to runs of 2 k."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat((b[:k], b[k:] + a[k:] * b[:-k]))
        a = torch.cat((a[:k], a[k:] * a[:-k]))
        k *= 2
    return b


def _memory(s):
    """(h, keep * a, the states before each step, ...) of a rollout in 32 bits."""
    x, gate = s['x'].detach().float(), s['gate'].detach().float()
    a, i = torch.sigmoid(gate), torch.sigmoid(-gate)
    ka = a if s['starts'] is None else torch.where(s['starts'].bool()[..., None], torch.zeros((), device=a.device), a)
    b = i * x
    if s['state'] is not None:
        b[0] += ka[0] * s['state'].detach()
    return x, a, i, ka, _scan(ka, b)


def _plain_step(s):
    x, gate = s['x'].float(), s['gate'].float()
    h = s['state'] if s['starts'] is None else torch.where(s['starts'].bool()[..., None], torch.zeros((), device=x.device), s['state'])
    h = torch.sigmoid(gate) * h + torch.sigmoid(-gate) * x
    return {'h': h.to(s['x'].dtype), 'state': h}


def _plain_scan(s):
    h = _memory(s)[-1]
    return {'h': h.to(s['x'].dtype), 'state': h[-1].clone()}


def _plain_train(s):
    x, a, i, ka, h = _memory(s)
    dt = s['x'].dtype
    first = torch.zeros_like(h[:1]) if s['state'] is None else s['state'].detach()[None]
    before = torch.cat((first, h[:-1]))
    if s['starts'] is not None:
        before = torch.where(s['starts'].bool()[..., None], torch.zeros((), device=a.device), before)
    grad = s['grad'].float().clone()
    grad[-1] += s['grad_state']
    back = torch.cat((torch.zeros_like(ka[:1]), ka.flip(0)[:-1]))
    lam = _scan(back, grad.flip(0)).flip(0)
    out = {'h': h.to(dt), 'state': h[-1].clone(), 'dx': (i * lam).to(dt), 'dgate': (lam * (before - x) * (a * i)).to(dt)}
    if s['state'] is not None:
        out['dstate'] = ka[0] * lam[0]
    return out


def _orthogonal(g):
    """Five Newton-Schulz steps on g / |g|, in g's type."""
    a, b, c = COEFFICIENTS
    turned = g.shape[-2] > g.shape[-1]
    x = g.transpose(-2, -1).contiguous() if turned else g
    norm = torch.sqrt((x * x).sum(dim=(-2, -1), keepdim=True))
    x = torch.where(norm > 0, x / norm, torch.zeros((), device=g.device, dtype=g.dtype))
    for _ in range(5):
        p = torch.matmul(x, x.transpose(-2, -1).contiguous())
        q = b * p + c * torch.matmul(p, p)
        x = a * x + torch.matmul(q, x)
    return x.transpose(-2, -1).contiguous() if turned else x


def _moved(w, g, m):
    """The weight update: momentum with look-ahead, orthogonalised, decoupled decay."""
    m = 0.95 * m + g
    o = _orthogonal(g + 0.95 * m)
    scale = math.sqrt(max(1.0, w.shape[-2] / w.shape[-1]))
    return (1.0 - 0.02 * 0.01) * w - 0.02 * scale * o, m


def _plain_orth(s):
    return {'o': _orthogonal(s['g'].float()).to(s['g'].dtype)}


def _plain_muon(s):
    w, m = _moved(s['w'].float(), s['g'].float(), s['m'])
    return {'w': w.to(s['w'].dtype), 'm': m}


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _own(s):
    op = s['case']['op']
    if op in ('orth', 'muon'):
        from drloco_amd import muon
        if op == 'orth':
            return {'o': muon.orthogonalise(s['g'])}
        w, m = muon.muon_update(s['w'], s['g'], s['m'], lr=0.02, beta=0.95, nesterov=True, weight_decay=0.01)
        return {'w': w, 'm': m}
    from drloco_amd import memory
    if op == 'step':
        h, state = memory.gated_memory_step(s['x'], s['gate'], s['state'], s['starts'])
        return {'h': h, 'state': state}
    h, state = memory.gated_memory(s['x'], s['gate'], s['starts'], s['state'])
    out = {'h': h, 'state': state}
    if op == 'train':
        leaves = [s['x'], s['gate']] + ([] if s['state'] is None else [s['state']])
        grads = torch.autograd.grad((h, state), leaves, (s['grad'], s['grad_state']))
        out.update(zip(('dx', 'dgate', 'dstate'), grads))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {'step': _plain_step, 'scan': _plain_scan, 'train': _plain_train, 'orth': _plain_orth, 'muon': _plain_muon}[state['case']['op']](state)


def work(case):
    e = torch.finfo(TYPES[case['type']]).bits // 8
    if case['op'] in ('orth', 'muon'):
        B, m, n = case['B'], min(case['m'], case['n']), max(case['m'], case['n'])
        # the gradient is read and the result written; the two symmetric products of a step need half their entries
        per = 2 * e if case['op'] == 'orth' else 3 * e + 8
        return {'bytes': B * m * n * per, 'flops': B * 5 * (m * m * n + m * m * m + 2 * m * m * n)}
    T, N, D = case['T'], case['N'], case['D']
    rows = T * N * (1 if case['every'] else 0) + N * D * (8 if case['state'] else 4)
    if case['op'] == 'train':          # x, gate and the gradient read; h, dx and dgate written
        return {'bytes': T * N * D * 6 * e + rows + N * D * (8 if case['state'] else 4), 'flops': T * N * D * 20}
    return {'bytes': T * N * D * 3 * e + rows, 'flops': T * N * D * 8}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case['op'] in ('orth', 'muon'):
            return _exact_update(case, s)
        return _exact_memory(case, s)


def _exact_update(case, s):
    g = s['g'].double()
    if case['op'] == 'muon':
        m = s['m'].double() * 0.95 + g
        g = g + 0.95 * m
    k1, k3, k5 = COEFFICIENTS
    out = []
    for y in (g if g.dim() == 3 else g[None]):
        y = y / y.norm() if float(y.norm()) > 0 else y
        for _ in range(5):          # k1 Y + k3 (Y Y') Y + k5 (Y Y')^2 Y, from the short side
            if y.shape[0] <= y.shape[1]:
                t = (y @ y.t()) @ y
                y = k1 * y + k3 * t + k5 * ((y @ y.t()) @ t)
            else:
                t = y @ (y.t() @ y)
                y = k1 * y + k3 * t + k5 * (t @ (y.t() @ y))
        out.append(y)
    o = torch.stack(out).reshape(s['g'].shape)
    if case['op'] == 'orth':
        return {'o': o}
    rows, cols = o.shape[-2:]
    return {'w': s['w'].double() * (1.0 - 0.02 * 0.01) - 0.02 * max(1.0, rows / cols) ** 0.5 * o, 'm': m}


def _exact_memory(case, s):
    T, N, D = case['T'], case['N'], case['D']
    x, g = s['x'].detach().double().reshape(T, N, D), s['gate'].detach().double().reshape(T, N, D)
    forget, take = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    if s['starts'] is None:
        keep = torch.ones(T, N, 1, dtype=torch.float64, device=x.device)
    else:
        keep = (s['starts'].reshape(T, N, 1) == 0).double()
    first = torch.zeros(N, D, dtype=torch.float64, device=x.device) if s['state'] is None else s['state'].detach().double()
    carried = forget * keep
    taken = take * x
    h = torch.empty_like(x)
    last = first
    for t in range(T):
        last = torch.addcmul(taken[t], carried[t], last, out=h[t])
    if case['op'] == 'step':
        return {'h': h[0], 'state': h[0].clone()}
    out = {'h': h, 'state': h[-1].clone()}
    if case['op'] == 'train':
        before = torch.cat((first[None], h[:-1])) * keep
        slope = (before - x) * forget * take
        dh = s['grad'].double()
        lam = s['grad_state'].double()
        zero = torch.zeros_like(lam)
        for t in range(T - 1, -1, -1):
            lam = torch.add(dh[t], lam, out=dh[t])
            lam = torch.addcmul(zero, carried[t], lam)
        out['dx'], out['dgate'] = take * dh, slope * dh
        if s['state'] is not None:
            out['dstate'] = lam
    return out
