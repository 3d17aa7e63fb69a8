"""Plain 64-bit restatements of the learner's operators, on the CPU, for tests/test_learner_*.py and tests/test_gpu_learner_*.py."""
import numpy as np


def memory(x, gate, starts=None, state=None):
    """h [T, N, D] and the last state, float64, step by step from the definition."""
    x, gate = np.asarray(x, np.float64), np.asarray(gate, np.float64)
    T, N, D = x.shape
    with np.errstate(over='ignore', invalid='ignore'):
        a, s = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
        h = np.zeros((T, N, D))
        last = np.zeros((N, D)) if state is None else np.asarray(state, np.float64).copy()
        for t in range(T):
            if starts is not None:
                last = np.where(np.asarray(starts[t], bool)[:, None], 0.0, last)
            last = a[t] * last + s[t] * x[t]
            h[t] = last
    return h, last


def memory_backward(x, gate, starts, state, grad_h, grad_last):
    """(dx, dgate, dstate, largest |gradient that reaches a step|) of sum(h grad_h) + sum(last grad_last), float64."""
    x, gate = np.asarray(x, np.float64), np.asarray(gate, np.float64)
    T, N, D = x.shape
    a, s = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
    h, _ = memory(x, gate, starts, state)
    lam = np.zeros((N, D)) if grad_last is None else np.asarray(grad_last, np.float64).copy()
    dx, dg, most = np.zeros_like(x), np.zeros_like(x), 0.0
    for t in range(T - 1, -1, -1):
        if grad_h is not None:
            lam = lam + np.asarray(grad_h[t], np.float64)
        most = max(most, np.nanmax(np.abs(lam), initial=0.0))
        before = h[t - 1] if t else (np.zeros((N, D)) if state is None else np.asarray(state, np.float64))
        keep = np.ones((N, 1)) if starts is None else 1.0 - np.asarray(starts[t], bool)[:, None]
        before = np.where(keep > 0, before, 0.0)
        dx[t] = s[t] * lam
        dg[t] = lam * (before - x[t]) * a[t] * s[t]
        lam = np.where(keep > 0, a[t] * lam, 0.0)
    return dx, dg, lam, most
