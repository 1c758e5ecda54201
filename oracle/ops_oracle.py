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


# ------------------------------------------------------------------ streams, symbols, linear attention
def rms_norm(total, weight=None, eps=1e-5):
    """(y, rstd) over the last axis of the stream as it was rounded."""
    total = f64(total)
    rstd = 1.0 / np.sqrt((total ** 2).mean(axis=-1) + eps)
    y = total * rstd[..., None]
    return (y if weight is None else y * f64(weight)), rstd


def rms_norm_backward(grad, total, weight=None, grad_total=None, eps=1e-5):
    """(dx, dweight): y_i = t_i w_i s^-1/2 with s = mean(t^2) + eps, so dy_i/dt_j = w_i (s^-1/2 [i = j] - t_i t_j s^-3/2 / n)."""
    grad, t = f64(grad), f64(total)
    s = (t ** 2).mean(axis=-1, keepdims=True) + eps
    h = grad if weight is None else grad * f64(weight)
    dx = h / np.sqrt(s) - t * (h * t).mean(axis=-1, keepdims=True) / s ** 1.5
    dweight = (grad * t / np.sqrt(s)).reshape(-1, t.shape[-1]).sum(axis=0)
    return (dx if grad_total is None else dx + f64(grad_total)), dweight


def embedding(table, tokens, scale=1.0):
    table, tokens = f64(table), np.asarray(tokens)
    known = (tokens >= 0) & (tokens < len(table))
    out = np.zeros((*tokens.shape, table.shape[1]))
    out[known] = scale * table[tokens[known]]
    return out


def embedding_backward(grad, tokens, rows, scale=1.0):
    grad, table = f64(grad), np.zeros((rows, np.shape(grad)[-1]))
    for token, g in zip(np.asarray(tokens).reshape(-1), grad.reshape(-1, grad.shape[-1])):
        if 0 <= token < rows:
            table[token] += scale * g
    return table


def counter_draw(seed, stream, tick, index):
    """The 64 bits whose upper 53 are the simulator's uniform draw."""
    mask = (1 << 64) - 1
    v = (seed ^ stream * 0x9E3779B97F4A7C15 ^ tick * 0xD1B54A32D192ED03 ^ index * 0x94D049BB133111EB) & mask
    v = ((v ^ v >> 30) * 0xBF58476D1CE4E5B9) & mask
    v = ((v ^ v >> 27) * 0x94D049BB133111EB) & mask
    return v ^ v >> 31


def dropout_kept(count, probability, seed, stream=0, tick=0):
    """Which of `count` values stay: 32 bits of a draw each, the low ones first."""
    draws = (counter_draw(seed, stream, tick, i // 2) >> (32 * (i % 2)) & 0xFFFFFFFF for i in range(count))
    threshold = min(int(probability * 2.0 ** 32 + 0.5), (1 << 32) - 1)
    return np.array([draw >= threshold for draw in draws], bool)


def _linear_inputs(q, k, v, log_decay, lengths):
    q, k, v = f64(q), f64(k), f64(v)
    group = v.shape[2] // q.shape[2]
    q, k = (np.repeat(a, group, axis=2) for a in (q, k))
    gates = v.shape[:3]
    decay = np.ones(gates) if log_decay is None else np.exp(np.broadcast_to(f64(log_decay), gates))
    live = np.ones(gates[:2], bool) if lengths is None else np.arange(gates[1]) < np.asarray(lengths)[:, None]
    return q, k, v, decay, live, group


def linear_attention(q, k, v, log_decay=None, state=None, lengths=None, scale=None):
    """(out, final state, states after each token) of S <- a S + k v^T, out = scale S^T q, token by token."""
    scale = np.shape(q)[-1] ** -0.5 if scale is None else scale
    q, k, v, decay, live, _ = _linear_inputs(q, k, v, log_decay, lengths)
    B, T, H, dk = q.shape
    S = np.zeros((B, H, dk, v.shape[-1])) if state is None else f64(state)
    out, states = np.zeros_like(v), np.zeros((T, *S.shape))
    for t in range(T):
        new = decay[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = np.where(live[:, t, None, None, None], new, S)
        out[:, t] = np.where(live[:, t, None, None], scale * (S * q[:, t, :, :, None]).sum(axis=2), 0.0)
        states[t] = S
    return out, S, states


def linear_attention_backward(grad_out, grad_state, q, k, v, log_decay=None, state=None, lengths=None, scale=None):
    """The gradients by the reversed recurrence, as a dict over the inputs."""
    scale = np.shape(q)[-1] ** -0.5 if scale is None else scale
    states, heads = linear_attention(q, k, v, log_decay, state, lengths, scale)[2], np.shape(q)[2]
    shared = log_decay is not None and np.ndim(log_decay) == 1
    q, k, v, decay, live, group = _linear_inputs(q, k, v, log_decay, lengths)
    do = f64(grad_out) * live[..., None, None] * scale
    B, T, H, dk = q.shape
    first = np.zeros_like(states[0]) if state is None else f64(state)
    D = np.zeros_like(states[0]) if grad_state is None else f64(grad_state)
    dq, dk_, dv, dg = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros((B, T, H))
    for t in reversed(range(T)):
        on = live[:, t, None, None]
        D = D + q[:, t, :, :, None] * do[:, t, :, None, :]
        dq[:, t] = (states[t] * do[:, t, :, None, :]).sum(axis=3)
        dk_[:, t] = np.where(on, (D * v[:, t, :, None, :]).sum(axis=3), 0.0)
        dv[:, t] = np.where(on, (D * k[:, t, :, :, None]).sum(axis=2), 0.0)
        faded = np.where(on[..., None], decay[:, t, :, None, None] * D, D)
        before = states[t - 1] if t else first
        dg[:, t] = np.where(on[..., 0], (faded * before).sum(axis=(2, 3)), 0.0)
        D = faded
    share = lambda a: a.reshape(B, T, heads, group, dk).sum(axis=3)  # noqa: E731
    return {"q": share(dq), "k": share(dk_), "v": dv, "log_decay": dg.sum(axis=(0, 1)) if shared else dg, "state": D}
