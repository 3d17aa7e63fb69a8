"""The gated memory of a recurrent policy: what a learner runs over the time-major rollout buffer next to the advantage scan, and
a policy in the loop runs once a control step.

    a[t] = sigmoid(gate[t])
    h[t] = a[t] * (0 if starts[t] else h[t-1]) + (1 - a[t]) * x[t]

x and gate are what the layer below computes from the observations; `starts` are the buffer's episode starts, as SB3's recurrent
buffers carry them (an episode that begins at t sees nothing of the one before).  The reference has no recurrent policy (its
CustomActorCriticPolicy, drloco/custom/policies.py:13-51, is a plain trunk); the operator stands where that trunk's hidden
layer stands, over the rollouts of drloco/train.py:110-118."""
import ctypes as C

import torch

from . import learner_lib as ll

_shape_ref = C.byref


def _rows(t):
    """t with a last axis that lies contiguously and walkers near enough for the kernels' 32-bit row offsets (any strides elsewhere)."""
    D = t.shape[-1]
    if t.stride(-1) != 1 and D > 1:
        return t.contiguous()
    if t.stride(-2) > 2000000 and t.shape[-2] > 1 and t.stride(-2) >= (1 << 29) // min(t.shape[-2], 256 // D + 2):
        return t.contiguous()
    return t


def _check(name, x, gate, starts, state, axes):
    for t in (x, gate, starts, state):
        if t is not None and not torch.is_tensor(t):
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
    ll.require_device(name, x, gate, starts, state)


def _shape(x, gate, starts, grad=None):
    s = ll.MemoryShape()
    s.T, s.N, s.D = x.shape
    s.x_t, s.x_n = x.stride()[:2]
    s.gate_t, s.gate_n = gate.stride()[:2]
    if starts is not None:
        s.starts_t, s.starts_n = starts.stride()
    if grad is not None:
        s.grad_t, s.grad_n = grad.stride()[:2]
    s.dtype = ll.DTYPES[x.dtype]
    return s


def _ptr(t):
    return None if t is None else t.data_ptr()


class _GatedMemory(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, starts, state):
        so = ll.load()
        T, N, D = x.shape
        with ll.on(x.device):
            s = _shape(x, gate, starts)
            h = torch.empty((T, N, D), dtype=x.dtype, device=x.device)
            last = torch.empty((N, D), dtype=torch.float32, device=x.device)
            wanted = any(ctx.needs_input_grad)
            marks = torch.empty((-(-T // ll.MARK), N, D), dtype=torch.float32, device=x.device) if wanted else None
            size = ll.check(so.dl_memory_workspace_bytes(_shape_ref(s)))
            work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
            ll.check(so.dl_memory_forward(_shape_ref(s), x.data_ptr(), gate.data_ptr(), _ptr(starts), _ptr(state), h.data_ptr(), last.data_ptr(), _ptr(marks), _ptr(work), ll.stream(x.device)))
        if wanted:
            ctx.save_for_backward(x, gate, starts, marks)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h, grad_last):
        if grad_h is None and grad_last is None:
            return None, None, None, None
        so = ll.load()
        x, gate, starts, marks = ctx.saved_tensors
        with ll.on(x.device):
            if grad_h is not None:
                grad_h = _rows(grad_h)
            if grad_last is not None:
                grad_last = grad_last.contiguous()
            s = _shape(x, gate, starts, grad_h)
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dgate = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dstate = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device) if ctx.needs_input_grad[3] else None
            size = ll.check(so.dl_memory_workspace_bytes(_shape_ref(s)))
            work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
            ll.check(so.dl_memory_backward(_shape_ref(s), x.data_ptr(), gate.data_ptr(), _ptr(starts), marks.data_ptr(), _ptr(grad_h), _ptr(grad_last), dx.data_ptr(), dgate.data_ptr(),
                                           _ptr(dstate), _ptr(work), ll.stream(x.device)))
        return dx, dgate, None, dstate


def gated_memory(x, gate, starts=None, state=None):
    """The memory over a rollout.  x, gate: [T, N, D] of one type (float32, bfloat16, float16) with any strides (a last axis that is
    not contiguous is copied); starts: uint8 or bool [T, N], nonzero = an episode begins at that step, or None; state: float32
    [N, D], the memory before the first step, or None for zeros.  Returns (h [T, N, D] of x's type, the state after the last step,
    float32 [N, D], unrounded).  Differentiable once with respect to x, gate and state.

    The memory is held and summed in float32 whatever the type of x; nothing before an episode's start is read, not even a NaN.
    An infinity within an episode makes that channel NaN until the next start.  T = 0 gives an empty h and the state as it came."""
    _check('gated_memory', x, gate, starts, state, 3)
    if x.numel() == 0:
        last = torch.zeros(x.shape[1:], dtype=torch.float32, device=x.device) if state is None else state.clone()
        return x.clone(), last
    x, gate = _rows(x), _rows(gate)
    if starts is not None and starts.dtype == torch.bool:
        starts = starts.view(torch.uint8)
    if state is not None:
        state = state.contiguous()
    return _GatedMemory.apply(x, gate, starts, state)


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


@torch.no_grad()
def gated_memory_step(x, gate, state, starts=None, out=None, state_out=None):
    """One control step of the memory, for a policy in the loop (no gradients): x, gate [N, D], state float32 [N, D], starts uint8 or
    bool [N] or None.  Returns (h [N, D] of x's type, the new state).  out / state_out: destinations (contiguous), e.g. a slot of
    the rollout buffer; state_out may be `state` itself; otherwise no argument overlaps a destination."""
    _check('gated_memory_step', x, gate, starts, state, 2)
    if state is None:
        raise TypeError('gated_memory_step: state must be a tensor')
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _destination('out', out, x, x.dtype, [t for t in (x, gate, state, starts) if t is not None])
    if state_out is None:
        state_out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    else:
        same = state_out is state or (state.is_contiguous() and state_out.data_ptr() == state.data_ptr())
        _destination('state_out', state_out, x, torch.float32, [t for t in (x, gate, out, starts) if t is not None] + ([] if same else [state]))
    if x.numel() == 0:
        return out, state_out
    x, gate = _rows(x), _rows(gate)
    state = state.contiguous()
    s = ll.MemoryShape()
    s.T, s.N, s.D = 1, x.shape[0], x.shape[1]
    s.x_n, s.gate_n = x.stride(0), gate.stride(0)
    if starts is not None:
        s.starts_n = starts.stride(0)
    s.dtype = ll.DTYPES[x.dtype]
    with ll.on(x.device):
        ll.check(ll.load().dl_memory_step(_shape_ref(s), x.data_ptr(), gate.data_ptr(), _ptr(starts), state.data_ptr(), out.data_ptr(), state_out.data_ptr(), ll.stream(x.device)))
    torch.autograd.graph.increment_version((out, state_out))          # the library wrote behind torch's back
    return out, state_out
