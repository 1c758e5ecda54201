"""The references of the stream, symbol and linear attention operators (oracle/ops_oracle.py), their C ABI and what they
refuse: everything that needs no GPU.  The references are pinned by torch autograd in float64 of separately written
forwards, by central differences and by the simulator's own draws."""
import ctypes
import inspect

import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo
from oracle import oracle


def linear_case(seed=0, B=2, T=9, H=2, Hv=4, dk=5, dv=3, shared=False):
    rng = np.random.default_rng(seed)
    return dict(q=rng.standard_normal((B, T, H, dk)), k=rng.standard_normal((B, T, H, dk)), v=rng.standard_normal((B, T, Hv, dv)),
                log_decay=-rng.random(Hv if shared else (B, T, Hv)), state=rng.standard_normal((B, Hv, dk, dv)))


def torch_linear(q, k, v, log_decay, state, scale):
    """All tokens at once: decayed scores, and the first state's share."""
    group, T = v.shape[2] // q.shape[2], q.shape[1]
    q, k = (a.repeat_interleave(group, dim=2) for a in (q, k))
    g = log_decay.expand(v.shape[:3]).cumsum(1)
    keep = torch.ones(T, T, dtype=torch.bool).tril()[None, :, :, None]
    decay = torch.exp((g[:, :, None] - g[:, None]).masked_fill(~keep, -torch.inf))
    out = scale * torch.einsum("bihk,bjhk,bijh,bjhv->bihv", q, k, decay, v)
    out = out + scale * torch.einsum("bihk,bih,bhkv->bihv", q, torch.exp(g), state)
    last = torch.einsum("bjhk,bjh,bjhv->bhkv", k, decay[:, -1], v) + torch.exp(g[:, -1])[..., None, None] * state
    return out, last


@pytest.mark.parametrize("shared", [False, True])
def test_linear_reference_matches_autograd(shared):
    case = linear_case(shared=shared)
    leaves = {n: torch.tensor(a, requires_grad=True) for n, a in case.items()}
    out, S = torch_linear(**leaves, scale=0.4)
    rng = np.random.default_rng(1)
    go, gs = rng.standard_normal(out.shape), rng.standard_normal(S.shape)
    got = oo.linear_attention(**case, scale=0.4)
    np.testing.assert_allclose(got[0], out.detach().numpy(), rtol=0, atol=1e-12)
    np.testing.assert_allclose(got[1], S.detach().numpy(), rtol=0, atol=1e-12)
    want = torch.autograd.grad([out, S], list(leaves.values()), [torch.tensor(go), torch.tensor(gs)])
    grads = oo.linear_attention_backward(go, gs, **case, scale=0.4)
    for name, g in zip(leaves, want):
        np.testing.assert_allclose(grads[name], g.numpy(), rtol=0, atol=1e-11, err_msg=name)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("lengths", [None, [9, 4], [0, 9]])
def test_linear_reference_matches_differences(lengths, shared):
    case = linear_case(3, shared=shared)
    rng = np.random.default_rng(4)
    go, gs = rng.standard_normal((2, 9, 4, 3)), rng.standard_normal((2, 4, 5, 3))

    def loss(c):
        out, S, _ = oo.linear_attention(**c, lengths=lengths)
        return float((out * go).sum() + (S * gs).sum())

    grads = oo.linear_attention_backward(go, gs, **case, lengths=lengths)
    for name in case:
        for flat in rng.choice(case[name].size, size=min(10, case[name].size), replace=False):
            at = np.unravel_index(flat, case[name].shape)
            pair = []
            for sign in (1, -1):
                moved = {n: a.copy() for n, a in case.items()}
                moved[name][at] += sign * 1e-6
                pair.append(loss(moved))
            difference = (pair[0] - pair[1]) / 2e-6
            assert abs(difference - grads[name][at]) <= 1e-7 + 1e-6 * abs(difference), (name, at)


def test_a_decay_gradient_taken_before_the_decay_is_caught(monkeypatch):
    """The gradient of log_decay with the state's gradient as it was before the token's decay."""
    right = "dg[:, t] = np.where(on[..., 0], (faded * before).sum(axis=(2, 3)), 0.0)"
    source = inspect.getsource(oo.linear_attention_backward)
    assert source.count(right) == 1
    planted = {}
    exec(source.replace(right, right.replace("faded", "D")), vars(oo), planted)
    monkeypatch.setattr(oo, "linear_attention_backward", planted["linear_attention_backward"])
    with pytest.raises(AssertionError, match="log_decay"):
        test_linear_reference_matches_autograd(False)
    with pytest.raises(AssertionError, match="log_decay"):
        test_linear_reference_matches_differences(None, False)


def test_rms_reference_matches_autograd():
    rng = np.random.default_rng(5)
    x, r, w, g, s = (rng.standard_normal((7, 11)) if i != 2 else rng.standard_normal(11) for i in range(5))
    leaves = [torch.tensor(a, requires_grad=True) for a in (x, r, w)]
    total = leaves[0] + leaves[1]
    y = torch.nn.functional.rms_norm(total, (11,), leaves[2], 1e-3)
    np.testing.assert_allclose(oo.rms_norm(x + r, w, 1e-3)[0], y.detach().numpy(), atol=1e-13)
    dx, dr, dw = torch.autograd.grad([y, total], leaves, [torch.tensor(g), torch.tensor(s)])
    got = oo.rms_norm_backward(g, x + r, w, s, 1e-3)
    for a, t in zip((got[0], got[0], got[1]), (dx, dr, dw)):
        np.testing.assert_allclose(a, t.numpy(), atol=1e-12)


def test_embedding_reference_matches_autograd():
    rng = np.random.default_rng(6)
    table, tokens = rng.standard_normal((5, 3)), np.array([[0, 4, 4, -1], [2, 4, 9, 0]])
    known = (tokens >= 0) & (tokens < 5)
    leaf = torch.tensor(table, requires_grad=True)
    out = 1.5 * torch.nn.functional.embedding(torch.tensor(np.where(known, tokens, 0)), leaf) * torch.tensor(known)[..., None]
    np.testing.assert_allclose(oo.embedding(table, tokens, 1.5), out.detach().numpy(), atol=1e-15)
    g = rng.standard_normal(out.shape)
    want, = torch.autograd.grad(out, leaf, torch.tensor(g))
    np.testing.assert_allclose(oo.embedding_backward(g, tokens, 5, 1.5), want.numpy(), atol=1e-14)


def test_draws_are_the_simulators():
    """The upper 53 bits of each draw are the simulator's uniform number of (seed, stream, tick, index)."""
    rng = np.random.default_rng(7)
    for _ in range(200):
        seed, stream, tick, index = (int(n) for n in rng.integers(0, 1 << 63, 4) >> rng.integers(0, 62, 4))
        assert (oo.counter_draw(seed, stream, tick, index) >> 11) * 2.0 ** -53 == oracle.counter_uniform(seed, stream, tick, index)


def test_dropped_shares():
    """Of 40000 values each share is met within five standard deviations, in either half of the draws; 0 drops none."""
    for p in (0.0, 0.1, 0.5, 0.9):
        kept = oo.dropout_kept(40000, p, 3, 1, 2)
        for half in (kept[::2], kept[1::2]):
            assert abs(half.mean() - (1 - p)) <= 5 * np.sqrt(p * (1 - p) / half.size)
    assert not np.array_equal(oo.dropout_kept(64, 0.5, 3, 1, 2), oo.dropout_kept(64, 0.5, 3, 1, 3))


# ------------------------------------------------------------------------------------------- the ABI
P = 4096  # an address that is never read: each call is refused


@pytest.fixture
def refused():
    lib, err = ops.library(), ctypes.create_string_buffer(256)

    def check(name, *args, text):
        rc = getattr(lib, name)(*args, None, ctypes.addressof(err), 256)
        assert rc == 7 and text in err.value.decode(), (name, rc, err.value)

    return check


def test_the_abi_refuses_streams_and_symbols(refused):
    rows = ops._ROWS.pack(P, 4, 0, 8)
    norm, back = "atlas_ops_rms_norm", "atlas_ops_rms_norm_backward"
    refused(norm, rows, None, 4, 0, 0, None, 0, 1e-5, P, None, None, None, text="width")
    refused(norm, rows, None, 4, 8, 2, None, 0, 1e-5, P, None, None, None, text="type")
    refused(norm, rows, None, 4, 8, 0, P, 1, 1e-5, P, None, None, None, text="type")
    refused(norm, None, None, 4, 8, 0, None, 0, 1e-5, P, None, None, None, text="null")
    refused(norm, rows, None, 4, 8, 0, None, 0, 1e-5, None, None, None, None, text="null")
    refused(norm, rows, rows, 4, 8, 0, None, 0, 1e-5, P, None, None, None, text="null")
    refused(norm, rows, None, 4, 8, 0, None, 0, 1e-5, P, None, P, None, text="null")
    refused(norm, rows, None, 1 << 24, 4100, 0, None, 0, 1e-5, P, None, None, None, text="2^24")
    refused(back, rows, rows, None, 4, 8, 0, None, 0, None, P, None, None, text="null")
    refused(back, rows, rows, None, 4, 8, 0, None, 0, P, P, P, None, text="null")
    refused(back, rows, rows, None, 1 << 24, 8200, 1, None, 0, P, P, P, P, text="2^24")
    look, sums = "atlas_ops_embedding", "atlas_ops_embedding_backward"
    refused(look, P, 0, 8, 8, 0, P, 0, 4, 1.0, P, text="positive")
    refused(look, P, 4, 0, 8, 0, P, 0, 4, 1.0, P, text="positive")
    refused(look, P, 4, 8, 8, 2, P, 0, 4, 1.0, P, text="type")
    refused(look, P, 4, 8, 8, 0, None, 0, 4, 1.0, P, text="null")
    refused(sums, rows, P, 0, 4, 4, 8, 2, 0, 1.0, P, P, text="type")
    refused(sums, rows, P, 0, 4, 4, 8, 0, 0, 1.0, None, P, text="null")
    refused(sums, None, P, 0, 4, 4, 8, 0, 0, 1.0, P, P, text="null")
    for count, table, width in ((-1, 4, 8), ((1 << 27) + 1, 4, 8), (4, 0, 8), (4, (1 << 31) - 1, 8), (4, 4, 0), (4, 4, (1 << 20) + 1)):
        refused(sums, rows, P, 0, count, table, width, 0, 0, 1.0, P, None, text="2^27")
        assert ops.library().atlas_ops_embedding_workspace(count, table, width, 0) == 0
    drop = "atlas_ops_dropout"
    refused(drop, P, None, 4, 2, 0.1, 0, 0, 0, None, P, text="type")
    for p in (-0.1, 1.0, 1.5, float("nan")):
        refused(drop, P, None, 4, 0, p, 0, 0, 0, None, P, text="probability")
    refused(drop, P, None, -1, 0, 0.1, 0, 0, 0, None, P, text="count")
    refused(drop, None, None, 4, 0, 0.1, 0, 0, 0, None, P, text="null")


def test_the_abi_refuses_linear_attention(refused):
    def linear(batch=1, time=1, heads=1, value_heads=1, key=4, value=4, type_=0, q=P, decay_type=0):
        return ops._DELTA.pack(q, P, P, P, 0, *([4] * 15), 0, 0, batch, time, heads, value_heads, key, value, type_, decay_type, 0, 1.0)

    lib = ops.library()
    for packed, text in ((linear(batch=0), "size"), (linear(key=0), "key"), (linear(key=129), "key"), (linear(value=129), "value"),
                         (linear(heads=2, value_heads=3), "multiple"), (linear(type_=2), "type"), (linear(decay_type=2), "type"),
                         (linear(batch=70000), "65535"), (linear(time=(1 << 29) + 1), "time"), (linear(q=0), "null")):
        refused("atlas_ops_linear_step", packed, P, P, text=text)
        refused("atlas_ops_linear_forward", packed, 0, P, P, P, text=text)
        refused("atlas_ops_linear_backward", packed, P, P, ops.struct.pack("@3q", 4, 4, 4), P, P, P, P, P, 0, P, P, text=text)
        assert lib.atlas_ops_linear_workspace(packed, 1) == lib.atlas_ops_linear_backward_workspace(packed) == 0
    refused("atlas_ops_linear_forward", linear(), 0, P, P, None, text="null")
    many = linear(batch=65535, value_heads=513)
    refused("atlas_ops_linear_forward", many, 0, P, P, P, text="2^25")
    without = ops._DELTA.pack(P, P, P, 0, 0, *([4] * 15), 0, 0, 1, 1, 1, 1, 4, 4, 0, 0, 0, 1.0)
    refused("atlas_ops_linear_backward", without, P, P, ops.struct.pack("@3q", 4, 4, 4), P, P, P, P, P, 0, P, P, text="decays")
    far = ops.struct.pack("@3q", 4, (1 << 24) + 1, 4)
    refused("atlas_ops_linear_backward", linear(), P, P, far, P, P, P, P, P, 0, P, P, text="2^24")
    apart = ops._DELTA.pack(P, P, P, P, 0, *([4, (1 << 24) + 1, 4] * 5), 0, 0, 1, 1, 1, 1, 4, 4, 0, 0, 0, 1.0)
    refused("atlas_ops_linear_forward", apart, 0, P, P, P, text="2^24")
    assert 0 < lib.atlas_ops_linear_workspace(linear(time=1000), 0) < lib.atlas_ops_linear_workspace(linear(time=1000), 1)


def test_tensors_on_the_cpu_are_refused():
    x, tokens = torch.zeros(2, 3, 2, 4), torch.zeros(2, 3, dtype=torch.int64)
    gate = torch.zeros(2, 3, 2)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm_8bit(x), lambda: ops.rms_norm_backward(x, x, None, gate),
                 lambda: ops.embedding(x[0, 0], tokens), lambda: ops.embedding_backward(x[:, :, 0], tokens, 4),
                 lambda: ops.dropout(x, 0.1, 0), lambda: ops.linear_attention(x, x, x, gate),
                 lambda: ops.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], gate[:, 0], torch.zeros(2, 2, 4, 4))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_what_may_share_memory_is_not_declared_apart():
    """Dropout's result may be its input or its residual: none of the kernel's pointers may promise otherwise."""
    source = (ops.LIBRARY.parent / "csrc" / "atlas_ops_symbols.hip").read_text()
    start = source.index("dropout_kernel(")
    assert "__restrict__" not in source[start:source.index("{", start)]
