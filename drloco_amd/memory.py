"""The gated memory of a recurrent policy: what a learner runs over the time-major rollout buffer next to the advantage scan, and
a policy in the loop runs once a control step.

    a[t] = sigmoid(gate[t])
    h[t] = a[t] * (0 if starts[t] else h[t-1]) + (1 - a[t]) * x[t]

x and gate are what the layer below computes from the observations; `starts` are the buffer's episode starts, as SB3's recurrent
buffers carry them (an episode that begins at t sees nothing of the one before).  The reference has no recurrent policy (its
CustomActorCriticPolicy, drloco/custom/policies.py:13-51, is a plain trunk); the operator stands where that trunk's hidden
layer stands, over the rollouts of drloco/train.py:110-118."""
import torch
from torch.autograd import forward_ad

from . import learner_lib as ll
from . import lib


def _check(name, x, gate, starts, state, axes, differentiable=False):
    for i, t in enumerate((x, gate, starts, state)):
        if not torch.is_tensor(t) and (i < 2 or t is not None):
            raise TypeError(f'{name}: expected tensors, got {type(t).__name__}')
    if x.dim() != axes:
        raise ValueError(f'{name}: x needs {axes} axes, got {tuple(x.shape)}')
    if gate.shape != x.shape:
        raise ValueError(f'{name}: gate {tuple(gate.shape)} is not of the shape of x {tuple(x.shape)}')
    if x.dtype not in ll.DTYPES:
        raise TypeError(f'{name}: x must be float32, bfloat16 or float16, got {x.dtype}')
    if gate.dtype != x.dtype:
        raise TypeError(f'{name}: gate is {gate.dtype}, x is {x.dtype}')
    if starts is not None:
        if starts.dtype not in (torch.uint8, torch.bool):
            raise TypeError(f'{name}: starts must be uint8 or bool, got {starts.dtype}')
        if starts.shape != x.shape[:-1]:
            raise ValueError(f'{name}: starts {tuple(starts.shape)} is not {tuple(x.shape[:-1])}')
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError(f'{name}: state must be float32, got {state.dtype}')
        if state.shape != x.shape[-2:]:
            raise ValueError(f'{name}: state {tuple(state.shape)} is not {tuple(x.shape[-2:])}')
    if differentiable and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, gate, state)):
        raise NotImplementedError(f'{name}: forward-mode derivatives are not supported')
    ll.require_device(name, x, gate, starts, state)


def gated_memory(x, gate, starts=None, state=None):
    """The memory over a rollout.  x, gate: [T, N, D] of one type (float32, bfloat16, float16) with any strides (a last axis that is
    not contiguous is copied); starts: uint8 or bool [T, N], nonzero = an episode begins at that step, or None; state: float32
    [N, D], the memory before the first step, or None for zeros.  Returns (h [T, N, D] of x's type, the state after the last step,
    float32 [N, D], unrounded).  Differentiable once with respect to x, gate and state, in reverse mode (forward-mode derivatives are refused).

    The memory is held and summed in float32 whatever the type of x; nothing before an episode's start is read, not even a NaN.
    An infinity within an episode leaves that channel infinite or NaN until the next start.  T = 0 gives an empty h and the state as it came."""
    out = ll.ops().gated_memory(x, gate, starts, state) if torch.is_tensor(x) and torch.is_tensor(gate) else None
    if out is None:
        _check('gated_memory', x, gate, starts, state, 3, differentiable=True)
        raise lib.DrlocoError('gated_memory: the arguments were refused')
    return out


def _extent(t):
    """First and last address of t's elements."""
    reach = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + reach * t.element_size()


def _overlap(a, b):
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 <= b1 and b0 <= a1


def _destination(name, t, x, dtype, apart):
    if not torch.is_tensor(t) or t.shape != x.shape or t.dtype != dtype or t.device != x.device or not t.is_contiguous():
        raise ValueError(f'gated_memory_step: {name} must be a contiguous {dtype} tensor of the shape {tuple(x.shape)} on {x.device}')
    if t.numel() and any(_overlap(t, o) for o in apart):
        raise ValueError(f'gated_memory_step: {name} overlaps another argument')
    return t


def gated_memory_step(x, gate, state, starts=None, out=None, state_out=None):
    """One control step of the memory, for a policy in the loop (no gradients): x, gate [N, D], state float32 [N, D], starts uint8 or
    bool [N] or None.  Returns (h [N, D] of x's type, the new state).  out / state_out: destinations (contiguous), e.g. a slot of
    the rollout buffer; state_out may be `state` itself; otherwise no argument overlaps a destination."""
    done = ll.ops().gated_memory_step(x, gate, state, starts, out, state_out) if torch.is_tensor(x) and torch.is_tensor(gate) and torch.is_tensor(state) else None
    if done is None:
        _check('gated_memory_step', x, gate, starts, state, 2)
        if state is None:
            raise TypeError('gated_memory_step: state must be a tensor')
        apart = [t for t in (x, gate, starts) if t is not None]
        if out is not None:
            _destination('out', out, x, x.dtype, apart + [state])
        if state_out is not None:
            same = state.is_contiguous() and state_out.data_ptr() == state.data_ptr()
            _destination('state_out', state_out, x, torch.float32, apart + [out] * (out is not None) + [state] * (not same))
        raise lib.DrlocoError('gated_memory_step: the arguments were refused')
    return done
