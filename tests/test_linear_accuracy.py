"""Linear attention over many chunks, held to what independent roundings leave: the results, and the gradients of the decays,
which the kernels sum anew from the states every eight chunks (256 tokens of float32, 512 of bfloat16).

Tolerances, relative to the norm of what is expected.  A state passes T / C chunks (C = 32 in float32, 64 in bfloat16) and is
rounded at most 14 times in each, relative to its own norm; what else a result passes (pieces, decays, a chunk's own products)
is within 20 more.  Independent roundings add as the root of the sum of their squares, and four standard deviations are allowed:
TOL = 4 sqrt(14 T / C + 20) 2^-24, 2e-6 to 6e-6.  A gradient takes two such states: twice that.  The sum of n tokens' gradients errs by
no more than sqrt(n) times the norm of their errors (Cauchy-Schwarz), whether they cancel or not.  Results of bfloat16 add
half a step of each value, 2^-8 of the norm.
"""
import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

F32, BF16 = torch.float32, torch.bfloat16
CHUNK, ANCHOR = {F32: 32, BF16: 64}, 8
CASES = [(1, 300, 2, 2, 32, 32), (1, 1000, 1, 2, 24, 16), (2, 650, 2, 4, 20, 24), (2, 1290, 2, 4, 20, 24), (1, 1290, 1, 1, 64, 128)]


def tolerance(T, dtype):
    return 4.0 * np.sqrt(14.0 * T / CHUNK[dtype] + 20.0) * 2.0 ** -24


def make(B, T, H, Hv, dk, dv, dtype, decay):
    """Inputs in float64 as the type holds them, and the gradients of the results."""
    g = torch.Generator().manual_seed(T + dk)
    normal = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    case = dict(q=normal(B, T, H, dk).to(dtype), k=(normal(B, T, H, dk) / dk ** 0.5).to(dtype), v=normal(B, T, Hv, dv).to(dtype),
                log_decay=-torch.exp(-6.0 + 6.0 * torch.rand((Hv,) if decay == "head" else (B, T, Hv), generator=g)), state=normal(B, Hv, dk, dv))
    return case, normal(B, T, Hv, dv).to(dtype), normal(B, Hv, dk, dv)


def wide(t):
    return t.double().cpu().numpy()


def per_token(case, go, gs):
    """The gradients with a decay that every token has for itself."""
    given = {n: wide(t) for n, t in case.items()}
    given["log_decay"] = np.broadcast_to(given["log_decay"], given["v"].shape[:3])
    return oo.linear_attention_backward(wide(go), wide(gs), **given)


def decay_error(got, want, tol):
    """The error of a gradient of decays, by token or by head, in parts of what `want`, by token, allows."""
    if got.ndim == 3:
        return np.linalg.norm(got - want) / (2 * tol * np.linalg.norm(want))
    n = want.shape[0] * want.shape[1]
    return (np.abs(got - want.sum(axis=(0, 1))) / (2 * tol * np.sqrt(n) * np.linalg.norm(want, axis=(0, 1)))).max()


def anchored(case, go, gs, every, carried=lambda decay, product: decay * product):
    """The gradient of log_decay by token as sums over the tokens behind within intervals of `every`, each of which starts from
    the product of the state and its gradient behind it."""
    a = {n: wide(t) for n, t in case.items()}
    q, k, v, decay, _, _ = oo._linear_inputs(a["q"], a["k"], a["v"], a["log_decay"], None)
    do = wide(go) * q.shape[-1] ** -0.5
    states, D = oo.linear_attention(**a)[2], wide(gs)
    T = q.shape[1]
    out = np.zeros(decay.shape)
    total = (states[-1] * D).sum(axis=(2, 3))
    for t in reversed(range(T)):
        if t < T - 1 and (t + 1) % every == 0:
            total = carried(decay[:, t + 1], (states[t] * D).sum(axis=(2, 3)))
        if t < T - 1:
            D = decay[:, t + 1, :, None, None] * D
        D = D + q[:, t, :, :, None] * do[:, t, :, None, :]
        total = total + (states[t] * q[:, t, :, :, None] * do[:, t, :, None, :]).sum(axis=(2, 3)) - (D * k[:, t, :, :, None] * v[:, t, :, None, :]).sum(axis=(2, 3))
        out[:, t] = total
    return out


@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", CASES)
def test_the_bound_tells_mistakes(sizes, dtype, decay):
    """In 64 bits the anchored sums are the reference's; none at all, and a carry that is left out or not decayed, are beyond the bound."""
    case, go, gs = make(*sizes, dtype, decay)
    want, every = per_token(case, go, gs)["log_decay"], ANCHOR * CHUNK[dtype]
    tol, whole = tolerance(sizes[1], dtype), (lambda g: g) if decay == "token" else (lambda g: g.sum(axis=(0, 1)))
    right = anchored(case, go, gs, every)
    np.testing.assert_allclose(right, want, rtol=0, atol=1e-9 * np.abs(want).max())
    assert decay_error(whole(right), want, tol) <= 1e-3
    assert decay_error(whole(0 * want), want, tol) > 10
    if sizes[1] > every:
        for carried in (lambda decay, product: 0.0 * product, lambda decay, product: product):
            assert decay_error(whole(anchored(case, go, gs, every, carried)), want, tol) > 10


@pytest.mark.gpu
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", CASES)
def test_results_and_gradients(sizes, dtype, decay):
    print(f"case: accuracy of linear attention {sizes} {dtype} {decay}", flush=True)
    case, go, gs = make(*sizes, dtype, decay)
    tol, rounded = tolerance(sizes[1], dtype), 2.0 ** -8 if dtype == BF16 else 0.0
    out, final, tape = ops.linear_attention(**{n: t.cuda() for n, t in case.items()}, tape=True)
    got = ops.linear_attention_backward(go.cuda(), gs.cuda(), tape)
    want = per_token(case, go, gs)
    wanted_out, wanted_final, _ = oo.linear_attention(**{n: wide(t) for n, t in case.items()})

    def error(x, expected, allowed):
        return np.linalg.norm(wide(x) - expected) / (allowed * np.linalg.norm(expected))

    errors = {"out": error(out, wanted_out, tol + rounded), "final": error(final, wanted_final, tol), "state": error(got["state"], want["state"], tol),
              **{n: error(got[n], want[n], 2 * tol + rounded) for n in "qkv"}, "log_decay": decay_error(wide(got["log_decay"]), want["log_decay"], tol)}
    print({n: round(float(e), 3) for n, e in errors.items()}, flush=True)
    assert all(e <= 1.0 for e in errors.values()), errors
