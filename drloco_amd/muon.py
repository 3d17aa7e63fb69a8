"""Orthogonalised weight updates for the learner: the Muon optimiser's update of a policy's weight matrices (Jordan et al. 2024) on
the matrix cores, next to the Adam steps the reference takes (drloco/train.py:110-118 builds SB3's PPO with it).

    orthogonalise(g)       the orthogonal factor of a gradient, by Newton-Schulz products
    muon_update(w, g, m)   momentum, orthogonalisation and the new weight in one call
    HipMuon                a torch optimiser of matrices built on it; vectors (biases, log_std) stay with Adam"""
import functools
import math

import torch

from . import learner_lib as ll

COEFFICIENTS = (3.4445, -4.7750, 2.0315)          # one step takes singular values in (0, 1] towards [0.7, 1.2], small ones 3.4-fold
CUBIC = (1.5, -0.5, 0.0)                          # the classic step: converges to 1, slowly from small singular values


def _matrix(name, what, t, dtypes):
    if not torch.is_tensor(t):
        raise TypeError(f'{name}: {what} must be a tensor, got {type(t).__name__}')
    if t.dim() < 2:
        raise ValueError(f'{name}: {what} needs at least two axes, got {tuple(t.shape)}')
    if t.dtype not in dtypes:
        raise TypeError(f'{name}: {what} is {t.dtype}, expected {" or ".join(str(d) for d in dtypes)}')


def _coefficients(name, steps, coefficients):
    if int(steps) != steps or not 1 <= steps <= 100:
        raise ValueError(f'{name}: steps must be 1 .. 100, got {steps}')
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f'{name}: coefficients must be three finite numbers, got {coefficients}')
    refused = _refused(int(steps), *(float(c) for c in coefficients))
    if refused:
        raise ValueError(f'{name}: {refused}, got {coefficients}')


@functools.lru_cache
def _refused(steps, a, b, c):
    L = ll.load()
    return L.dl_learner_last_error().decode() if L.dl_orth_check_coefficients(steps, a, b, c) < 0 else None


def _result(name, what, t, like, dtype, aliases):
    """A destination given by the caller: the shape of `like`, contiguous; it is one of `aliases` or overlaps none of them."""
    if not torch.is_tensor(t) or t.shape != like.shape or t.dtype != dtype or t.device != like.device or not t.is_contiguous():
        raise ValueError(f'{name}: {what} must be a contiguous {dtype} tensor of shape {tuple(like.shape)} on {like.device}')
    lo, hi = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    for may, o in aliases:
        if o is None or not o.numel() or not t.numel():
            continue
        reach = sum((n - 1) * st for n, st in zip(o.shape, o.stride()))
        o0, o1 = o.data_ptr(), o.data_ptr() + (reach + 1) * o.element_size()
        if lo < o1 and o0 < hi and not (may and o0 == lo and o.is_contiguous() and o.dtype == dtype):
            raise ValueError(f'{name}: {what} overlaps another argument')
    return t


def orthogonalise(g, steps=5, coefficients=COEFFICIENTS, out=None):
    """The orthogonal factor U V' of each matrix G = U S V' of g [..., rows, cols] (float32, bfloat16 or float16), approached by `steps`
    steps X <- a X + b (X X') X + c (X X')^2 X from G / |G|_F: singular values move towards one, zeros and a zero matrix
    stay zero.  A matrix that holds a NaN or an infinity becomes NaN, the others of the batch do not.  Returns a tensor like g, or writes `out` (which
    may be g).  Not differentiable: it makes an update, not an activation.

    Operands are held to 22 bits (short sides of up to 16 next to long ones of up to 130560: to 32 in all products but X X') and summed in 32, for every type
    of g; a 16-bit result is the float32 one rounded.  A step multiplies what is lost in the directions of small singular values by a, five steps by 485.  Coefficients that let X, X X' or a + b X X' + c (X X')^2
    grow to 60 or more (default ones: 3.5) are refused."""
    _matrix('orthogonalise', 'g', g, tuple(ll.DTYPES))
    _coefficients('orthogonalise', steps, coefficients)
    ll.require_device('orthogonalise', g, out)
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    else:
        _result('orthogonalise', 'out', out, g, g.dtype, [(True, g)])
    if g.numel():
        ll.ops().orth_update(g, None, None, None, out, int(steps), *coefficients, 0.0, False, 0.0, 1.0)
    return out


def muon_update(weight, grad, momentum, lr, beta=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5, coefficients=COEFFICIENTS, out=None, momentum_out=None):
    """One step of the Muon optimiser for the matrices weight [..., rows, cols] (float32, bfloat16 or float16) with gradient `grad` (one of
    these types too) and momentum (float32):

        momentum' = beta momentum + grad,   u = grad + beta momentum' (nesterov) or momentum'
        weight'   = (1 - lr weight_decay) weight - lr scale orthogonalise(u)          scale: sqrt(max(1, rows / cols)) unless given

    computed in float32 (orthogonalise has more to say on it) and rounded once.  Returns (weight', momentum').  out / momentum_out:
    destinations (contiguous), e.g. weight and momentum themselves for an update in place."""
    name = 'muon_update'
    _matrix(name, 'weight', weight, tuple(ll.DTYPES))
    _matrix(name, 'grad', grad, tuple(ll.DTYPES))
    _matrix(name, 'momentum', momentum, (torch.float32,))
    for what, t in (('grad', grad), ('momentum', momentum)):
        if t.shape != weight.shape:
            raise ValueError(f'{name}: {what} {tuple(t.shape)} is not of the shape of weight {tuple(weight.shape)}')
    _coefficients(name, steps, coefficients)
    ll.require_device(name, weight, grad, momentum, out, momentum_out)
    if momentum_out is None:
        momentum_out = torch.empty(momentum.shape, dtype=torch.float32, device=momentum.device)
    else:
        _result(name, 'momentum_out', momentum_out, momentum, torch.float32, [(True, momentum), (False, weight), (False, grad)])
    if out is None:
        out = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
    else:
        _result(name, 'out', out, weight, weight.dtype, [(True, weight), (True, grad), (False, momentum), (False, momentum_out)])
    if scale is None:
        scale = math.sqrt(max(1.0, weight.shape[-2] / max(1, weight.shape[-1])))
    if weight.numel():
        ll.ops().orth_update(grad, momentum, momentum_out, weight, out, int(steps), *coefficients, beta, bool(nesterov), 1.0 - lr * weight_decay, -lr * scale)
    return out, momentum_out


class HipMuon(torch.optim.Optimizer):
    """Muon for the weight matrices of a policy, each step one muon_update in place per matrix.  Parameters need at least two axes, contiguous,
    on a HIP device; of more than two axes the last two are the matrices, the others a stack of them (for a convolution's weight, give a [out, rest] parameter); everything else (biases, log_std, usually the first and the last layer) belongs to another optimiser.
    With walkers sharded over GPUs the gradients are summed over the ranks first (collectives.FlatGradAllReducer); every rank then takes the same step.
    step() can be captured into a graph after a first eager one; a replay takes the learning rate that was set at the capture."""

    def __init__(self, params, lr=0.02, beta=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS):
        if not lr >= 0.0 or not weight_decay >= 0.0 or not 0.0 <= beta < 1.0:
            raise ValueError(f'HipMuon: lr {lr}, weight_decay {weight_decay} or beta {beta} out of range')
        _coefficients('HipMuon', steps, coefficients)
        super().__init__(params, dict(lr=lr, beta=beta, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=tuple(coefficients)))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]['params']:
            if p.dim() < 2 or p.dtype not in ll.DTYPES or not p.is_contiguous():
                bad = self.param_groups.pop()
                raise ValueError(f'HipMuon: parameters must be contiguous matrices of float32, bfloat16 or float16, got {tuple(p.shape)} {p.dtype} among {len(bad["params"])}')

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError('HipMuon: sparse gradients are not supported')
                state = self.state[p]
                if not state:
                    if torch.cuda.is_current_stream_capturing():          # (every replay would begin with no momentum)
                        raise RuntimeError('HipMuon: the first step makes the momenta: take it before it is captured into a graph')
                    state['momentum'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                muon_update(p, p.grad, state['momentum'], lr=float(group['lr']), beta=group['beta'], nesterov=group['nesterov'], weight_decay=group['weight_decay'],
                            steps=group['steps'], coefficients=group['coefficients'], out=p, momentum_out=state['momentum'])
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, with the momenta in float32 whatever the type of the weights (torch casts state to the parameter's type)."""
        super().load_state_dict(state_dict)
        saved = [k for g in state_dict['param_groups'] for k in g['params']]
        mine = [p for g in self.param_groups for p in g['params']]
        for k, p in zip(saved, mine):
            if k in state_dict['state'] and 'momentum' in state_dict['state'][k]:
                self.state[p]['momentum'] = state_dict['state'][k]['momentum'].to(device=p.device, dtype=torch.float32).clone().contiguous()
