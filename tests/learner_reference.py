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


def orthogonal(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), trace=None):
    """float64 [..., rows, cols]: `steps` Newton-Schulz steps from g / |g|.  trace: a list that takes |X|_F of every iterate."""
    g = np.asarray(g, np.float64)
    a, b, c = coefficients
    out = np.empty_like(g)
    for at in np.ndindex(g.shape[:-2]):
        x = g[at]
        turned = x.shape[0] > x.shape[1]
        x = x.T if turned else x
        norm = np.sqrt((x * x).sum())
        x = x / norm if norm != 0 else x
        for _ in range(steps):
            if trace is not None:
                trace.append(np.sqrt((x * x).sum()))
            p = x @ x.T
            x = a * x + (b * p + c * (p @ p)) @ x
        out[at] = x.T if turned else x
    return out


def muon(w, g, m, lr, beta=0.95, nesterov=True, weight_decay=0.0, scale=None, **kw):
    """(new weight, new momentum), float64"""
    w, g, m = (np.asarray(t, np.float64) for t in (w, g, m))
    m = beta * m + g
    o = orthogonal(g + beta * m if nesterov else m, **kw)
    scale = np.sqrt(max(1.0, w.shape[-2] / w.shape[-1])) if scale is None else scale
    return (1 - lr * weight_decay) * w - lr * scale * o, m
