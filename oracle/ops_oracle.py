"""Float64 reference of the sequence-layer operators (NumPy, one token or one row at a time).

Written from the definitions, apart from the kernels' formulation: the delta rule runs its recurrence
token by token and its gradients are the reversed recurrence over stored states, where the kernels
work in chunks.  Inputs of any float type are widened first.
"""
from __future__ import annotations

import numpy as np


def f64(a):
    return None if a is None else np.asarray(a, np.float64)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) over the last axis."""
    x = f64(x)
    mean = x.mean(axis=-1)
    rstd = 1.0 / np.sqrt(((x - mean[..., None]) ** 2).mean(axis=-1) + eps)
    y = (x - mean[..., None]) * rstd[..., None]
    if weight is not None:
        y = y * f64(weight)
    return (y if bias is None else y + f64(bias)), mean, rstd


def layer_norm_backward(grad, x, weight=None, eps=1e-5):
    """(dx, dweight, dbias): the Jacobian of one row, row by row, then the sums over rows."""
    grad, x = f64(grad), f64(x)
    z, _, rstd = layer_norm(x, eps=eps)
    h = grad if weight is None else grad * f64(weight)
    dx = rstd[..., None] * (h - h.mean(axis=-1, keepdims=True) - z * (h * z).mean(axis=-1, keepdims=True))
    width = x.shape[-1]
    return dx, (grad * z).reshape(-1, width).sum(axis=0), grad.reshape(-1, width).sum(axis=0)


def orthogonalize(matrix, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Through the singular values: each step maps s to a s + b s^3 + c s^5 and keeps the singular vectors."""
    u, s, vt = np.linalg.svd(f64(matrix), full_matrices=False)
    a, b, c = coefficients
    s = s / (np.sqrt((s ** 2).sum(axis=-1, keepdims=True)) + eps)
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return (u * s[..., None, :]) @ vt


def muon(weight, gradient, momentum, *, learning_rate, factor=0.95, weight_decay=0.0, nesterov=True, scale=None, **kw):
    """(weight, momentum) after one step."""
    weight, gradient = f64(weight), f64(gradient)
    momentum = factor * f64(momentum) + gradient
    update = orthogonalize(gradient + factor * momentum if nesterov else momentum, **kw)
    if scale is None:
        scale = np.sqrt(max(1.0, weight.shape[-1] / weight.shape[-2]))
    return (1.0 - learning_rate * weight_decay) * weight - learning_rate * scale * update, momentum


def delta_rule(q, k, v, log_decay, beta, state=None, lengths=None, scale=None):
    """(out, final state, states before each token) of the recurrence."""
    q, k, v, beta = f64(q), f64(k), f64(v), f64(beta)
    B, T, H, dk = q.shape
    Hv, dv = v.shape[2:]
    scale = dk ** -0.5 if scale is None else scale
    S = np.zeros((B, Hv, dk, dv)) if state is None else f64(state).copy()
    out, states = np.zeros((B, T, Hv, dv)), np.zeros((T, B, Hv, dk, dv))
    for t in range(T):
        states[t] = S
        for b in range(B):
            if lengths is not None and t >= lengths[b]:
                continue
            for h in range(Hv):
                kt, qt = k[b, t, h // (Hv // H)], q[b, t, h // (Hv // H)]
                if log_decay is not None:
                    S[b, h] = S[b, h] * np.exp(np.float64(log_decay[b, t, h]))
                S[b, h] += beta[b, t, h] * np.outer(kt, v[b, t, h] - kt @ S[b, h])
                out[b, t, h] = scale * (qt @ S[b, h])
    return out, S, states


def delta_rule_backward(grad_out, grad_state, q, k, v, log_decay, beta, state=None, lengths=None, scale=None):
    """The gradients by the reversed recurrence, as a dict over the inputs."""
    states = delta_rule(q, k, v, log_decay, beta, state, lengths, scale)[2]
    q, k, v, beta, grad_out = f64(q), f64(k), f64(v), f64(beta), f64(grad_out)
    B, T, H, dk = q.shape
    Hv, dv = v.shape[2:]
    scale = dk ** -0.5 if scale is None else scale
    dS = np.zeros((B, Hv, dk, dv)) if grad_state is None else f64(grad_state).copy()
    g = {"q": np.zeros_like(q), "k": np.zeros_like(k), "v": np.zeros_like(v), "log_decay": np.zeros((B, T, Hv)),
         "beta": np.zeros((B, T, Hv))}
    for t in reversed(range(T)):
        for b in range(B):
            if lengths is not None and t >= lengths[b]:
                continue
            for h in range(Hv):
                hk = h // (Hv // H)
                kt, qt, bt, do = k[b, t, hk], q[b, t, hk], beta[b, t, h], scale * grad_out[b, t, h]
                a = 1.0 if log_decay is None else np.exp(np.float64(log_decay[b, t, h]))
                faded = a * states[t, b, h]
                e = v[b, t, h] - kt @ faded
                after = faded + bt * np.outer(kt, e)
                D = dS[b, h] + np.outer(qt, do)
                g["q"][b, t, hk] += after @ do
                g["beta"][b, t, h] = kt @ D @ e
                de = bt * (kt @ D)
                g["v"][b, t, h] = de
                g["k"][b, t, hk] += bt * (D @ e) - faded @ de
                D = D - np.outer(kt, de)
                g["log_decay"][b, t, h] = (D * faded).sum()
                dS[b, h] = a * D
    g["state"] = dS
    return g
