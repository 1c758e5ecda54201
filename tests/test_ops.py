"""The sequence-layer operators' reference (oracle/ops_oracle.py), their C ABI and what they refuse:
everything that needs no GPU.  The reference is pinned by torch autograd in float64 of separately written
forwards and by central differences."""
import ctypes
import inspect
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "operators" / "atlas_ops.h"


def delta_case(seed=0, B=2, T=9, H=2, Hv=4, dk=5, dv=3):
    rng = np.random.default_rng(seed)
    q, k = (rng.standard_normal((B, T, H, dk)) for _ in range(2))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    return dict(q=q, k=k, v=rng.standard_normal((B, T, Hv, dv)), log_decay=-rng.random((B, T, Hv)),
                beta=rng.random((B, T, Hv)), state=rng.standard_normal((B, Hv, dk, dv)))


def torch_delta(q, k, v, log_decay, beta, state, scale):
    group = v.shape[2] // q.shape[2]
    q, k = (a.repeat_interleave(group, dim=2) for a in (q, k))
    out, S = [], state
    for t in range(q.shape[1]):
        S = S * torch.exp(log_decay[:, t])[..., None, None]
        e = v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t])
        S = S + torch.einsum("bhk,bhv->bhkv", k[:, t] * beta[:, t][..., None], e)
        out.append(scale * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    return torch.stack(out, dim=1), S


def test_delta_reference_matches_autograd():
    case = delta_case()
    leaves = {n: torch.tensor(a, requires_grad=True) for n, a in case.items()}
    out, S = torch_delta(**leaves, scale=0.4)
    rng = np.random.default_rng(1)
    go, gs = rng.standard_normal(out.shape), rng.standard_normal(S.shape)
    got = oo.delta_rule(*case.values(), scale=0.4)
    np.testing.assert_allclose(got[0], out.detach().numpy(), rtol=0, atol=1e-13)
    np.testing.assert_allclose(got[1], S.detach().numpy(), rtol=0, atol=1e-13)
    want = torch.autograd.grad([out, S], list(leaves.values()), [torch.tensor(go), torch.tensor(gs)])
    grads = oo.delta_rule_backward(go, gs, *case.values(), scale=0.4)
    for name, g in zip(leaves, want):
        np.testing.assert_allclose(grads[name], g.numpy(), rtol=0, atol=1e-12, err_msg=name)


@pytest.mark.parametrize("lengths", [None, [9, 4], [0, 9]])
def test_delta_reference_matches_differences(lengths):
    case = delta_case(3)
    rng = np.random.default_rng(4)
    go, gs = rng.standard_normal((2, 9, 4, 3)), rng.standard_normal((2, 4, 5, 3))

    def loss(c):
        out, S, _ = oo.delta_rule(*c.values(), lengths=lengths)
        return float((out * go).sum() + (S * gs).sum())

    grads = oo.delta_rule_backward(go, gs, *case.values(), lengths=lengths)
    for name in case:
        for flat in rng.choice(case[name].size, size=10, replace=False):
            at = np.unravel_index(flat, case[name].shape)
            pair = []
            for sign in (1, -1):
                moved = {n: a.copy() for n, a in case.items()}
                moved[name][at] += sign * 1e-6
                pair.append(loss(moved))
            difference = (pair[0] - pair[1]) / 2e-6
            assert abs(difference - grads[name][at]) <= 1e-7 + 1e-6 * abs(difference), (name, at)


def test_norm_reference_matches_autograd():
    rng = np.random.default_rng(5)
    x, w, b, g = rng.standard_normal((7, 11)), rng.standard_normal(11), rng.standard_normal(11), rng.standard_normal((7, 11))
    leaves = [torch.tensor(a, requires_grad=True) for a in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (11,), leaves[1], leaves[2], 1e-3)
    np.testing.assert_allclose(oo.layer_norm(x, w, b, 1e-3)[0], y.detach().numpy(), atol=1e-13)
    want = torch.autograd.grad(y, leaves, torch.tensor(g))
    for a, t in zip(oo.layer_norm_backward(g, x, w, 1e-3), want):
        np.testing.assert_allclose(a, t.numpy(), atol=1e-12)


def test_orthogonal_reference_matches_products():
    rng = np.random.default_rng(6)
    a, b, c = ops.COEFFICIENTS
    for shape in ((5, 9), (9, 5), (3, 6, 6), (1, 4)):
        m = rng.standard_normal(shape)
        x = m / (np.sqrt((m ** 2).sum(axis=(-2, -1), keepdims=True)) + 1e-7)
        for _ in range(5):
            g = x @ np.swapaxes(x, -1, -2)
            x = a * x + (b * g + c * g @ g) @ x
        np.testing.assert_allclose(oo.orthogonalize(m), x, atol=1e-11)


def test_header_declares_what_the_library_exports():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = re.findall(r"^\s*(?:int|int64_t)\s+(\w+)\s*\(", text, flags=re.M)
    assert sorted(declared) == sorted(ops.EXPORTS)
    lib = ops.library()
    assert all(hasattr(lib, name) for name in declared)


def test_packed_structures_match_the_header():
    """Each struct's fields in the header, sized as a C compiler lays them out, against the packed layout."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    kinds = {"int64_t": ctypes.c_int64, "int": ctypes.c_int, "float": ctypes.c_float}
    for name, packed in (("AtlasRows", ops._ROWS), ("AtlasOrthogonal", ops._ORTHOGONAL), ("AtlasDelta", ops._DELTA)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
        fields = []
        for line in filter(None, (s.strip() for s in body.split(";"))):
            base, rest = re.match(r"((?:const\s+)?\w+)\s*(.*)", line, flags=re.S).groups()
            for item in rest.split(","):
                item = item.strip()
                kind = ctypes.c_void_p if item.startswith("*") else kinds[base]
                count = re.search(r"\[(\d+)\]", item)
                fields.append((item.strip("* "), kind * int(count.group(1)) if count else kind))
        struct_type = type(name, (ctypes.Structure,), {"_fields_": fields})
        codes = re.findall(r"(\d*)([Pqif])", packed.format)
        flat = [c for n, c in codes for _ in range(int(n or 1))]
        want = []
        for _, kind in fields:
            one, n = (kind._type_, kind._length_) if hasattr(kind, "_length_") else (kind, 1)
            want += [{ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int: "i", ctypes.c_float: "f"}[one]] * n
        assert flat == want, name
        assert packed.size <= ctypes.sizeof(struct_type) < packed.size + 8, name


def test_the_abi_refuses_before_it_launches():
    lib = ops.library()
    err = ctypes.create_string_buffer(256)
    address = ctypes.addressof(err)
    p = 4096  # never read: each call is refused
    rows = ops._ROWS.pack(p, 4, 0, 8)

    def refused(rc, text):
        assert rc == 7 and text in err.value.decode(), err.value

    refused(lib.atlas_ops_layer_norm(rows, 4, 0, 0, None, None, 0, 1e-5, p, None, None, None, address, 256), "width")
    refused(lib.atlas_ops_layer_norm(rows, 4, 8, 2, None, None, 0, 1e-5, p, None, None, None, address, 256), "type")
    refused(lib.atlas_ops_layer_norm(rows, 4, 8, 0, p, None, 1, 1e-5, p, None, None, None, address, 256), "type")
    refused(lib.atlas_ops_layer_norm(None, 4, 8, 0, None, None, 0, 1e-5, p, None, None, None, address, 256), "null")
    refused(lib.atlas_ops_layer_norm(rows, 4, 8, 0, None, None, 0, 1e-5, None, None, None, None, address, 256), "null")
    refused(lib.atlas_ops_layer_norm(rows, 4, 8, 0, None, None, 0, 1e-5, p, p, None, None, address, 256), "null")
    refused(lib.atlas_ops_layer_norm_backward(rows, rows, 4, 8, 0, None, 0, None, p, p, p, p, p, None, address, 256), "null")
    refused(lib.atlas_ops_layer_norm_backward(rows, rows, 4, 8, 0, None, 0, p, p, p, p, p, None, None, address, 256), "null")

    def orthogonal(batch=1, rows_=4, columns=4, out=p, weight=0, type_=0, steps=5):
        return ops._ORTHOGONAL.pack(p, batch, rows_, columns, 16, 4, 0, out, weight, type_, 0, 1, steps, 0.9, 1e-7, 1.0, 0.1,
                                    3.0, -4.0, 2.0)

    for packed, text in ((orthogonal(out=0), "null"), (orthogonal(weight=p), "null"), (orthogonal(batch=0), "batch"),
                         (orthogonal(steps=0), "steps"), (orthogonal(steps=65), "steps"), (orthogonal(type_=3), "type"),
                         (orthogonal(rows_=17000, columns=17000), "16384"), (orthogonal(rows_=1 << 21), "rows")):
        refused(lib.atlas_ops_orthogonalize(packed, p, None, address, 256), text)

    def delta(batch=1, time=1, heads=1, value_heads=1, key=4, value=4, type_=0, beta=p):
        return ops._DELTA.pack(p, p, p, p, beta, *([4] * 15), 0, 0, batch, time, heads, value_heads, key, value, type_,
                               0, 0, 1.0)

    for packed, text in ((delta(batch=0), "size"), (delta(key=0), "key"), (delta(key=129), "key"),
                         (delta(heads=2, value_heads=3), "multiple"), (delta(type_=2), "type"), (delta(beta=0), "null"),
                         (delta(batch=70000), "65535"), (delta(time=1 << 31), "time"), (delta(value=1 << 21), "value")):
        refused(lib.atlas_ops_delta_step(packed, p, p, None, address, 256), text)
        refused(lib.atlas_ops_delta_forward(packed, 0, p, p, p, None, address, 256), text)
        assert lib.atlas_ops_delta_workspace(packed, 1) == 0
    refused(lib.atlas_ops_delta_forward(delta(), 0, p, p, None, None, address, 256), "null")


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(2, 3, 2, 4)
    gate = torch.zeros(2, 3, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.layer_norm(x)
    with pytest.raises(ValueError, match="GPU"):
        ops.orthogonalize(x[0, 0])
    with pytest.raises(ValueError, match="GPU"):
        ops.muon_update(x[0, 0], x[0, 0], x[0, 0], learning_rate=0.1)
    with pytest.raises(ValueError, match="GPU"):
        ops.delta_rule(x, x, x, gate, gate)
    with pytest.raises(ValueError, match="GPU"):
        ops.delta_rule_step(x[:, 0], x[:, 0], x[:, 0], gate[:, 0], gate[:, 0], torch.zeros(2, 2, 4, 4))


def test_planted_mistake_in_the_reference_is_caught(monkeypatch):
    """The decay's gradient taken after the correction's write instead of before it."""
    case = delta_case(7)
    go = np.random.default_rng(8).standard_normal((2, 9, 4, 3))
    right = oo.delta_rule_backward(go, None, *case.values())["log_decay"]
    original = np.exp
    monkeypatch.setattr(oo.np, "exp", lambda a: original(a) * 1.001)
    wrong = oo.delta_rule_backward(go, None, *case.values())["log_decay"]
    assert np.abs(right - wrong).max() > 1e-4


def test_workspace_sizes():
    lib = ops.library()
    packed = ops._DELTA.pack(1, 1, 1, 1, 1, *([4] * 15), 0, 0, 2, 65, 2, 4, 5, 17, 0, 0, 0, 1.0)
    assert lib.atlas_ops_delta_workspace(packed, 0) > 0
    assert lib.atlas_ops_delta_workspace(packed, 1) > lib.atlas_ops_delta_workspace(packed, 0)
    assert lib.atlas_ops_delta_backward_workspace(packed) > 0
    assert lib.atlas_ops_layer_norm_workspace(1000, 256, 0) > 0 and lib.atlas_ops_layer_norm_workspace(0, 256, 0) == 0
    assert lib.atlas_ops_orthogonalize_workspace(1, 100, 50) > 0


def test_the_abi_refuses_what_a_launch_could_not_take():
    """A grid holds fewer than 2^32 threads along x: more is an invalid argument, not a failed launch.  A refused size
    has no workspace, and is refused for its size before the workspace is asked for."""
    lib = ops.library()
    err = ctypes.create_string_buffer(256)
    address = ctypes.addressof(err)
    p = 4096  # never read: each call is refused

    def refused(rc, text):
        assert rc == 7 and text in err.value.decode(), (rc, err.value)

    def delta(batch, time, value_heads, key, value):
        return ops._DELTA.pack(p, p, p, p, p, *([4] * 15), 0, 0, batch, time, 1, value_heads, key, value, 0, 0, 0, 1.0)

    # 65535 x 17 heads of 128 columns: 8 slices of 512 threads for each, of 256 with keys of 64; 2^29 + 1 tokens: more
    # than 2^23 chunks of 512 threads
    for packed, text in ((delta(65535, 64, 17, 128, 128), "value_heads x value"), (delta(65535, 64, 33, 64, 128), "value_heads x value"),
                         (delta(1, (1 << 29) + 1, 1, 16, 16), "time")):
        refused(lib.atlas_ops_delta_forward(packed, 0, p, p, p, None, address, 256), text)
        refused(lib.atlas_ops_delta_backward(packed, p, p, ops.struct.pack("@3q", 4, 4, 4), p, p, p, p, p, p, p, p, None,
                                             address, 256), text)
        assert lib.atlas_ops_delta_workspace(packed, 0) == lib.atlas_ops_delta_workspace(packed, 1) == 0
        assert lib.atlas_ops_delta_backward_workspace(packed) == 0
    assert lib.atlas_ops_delta_workspace(delta(65535, 64, 16, 128, 128), 0) > 0
    assert lib.atlas_ops_delta_workspace(delta(1, (1 << 29) - 64, 1, 16, 16), 0) > 0

    rows = ops._ROWS.pack(p, 1 << 24, 0, 8)
    assert lib.atlas_ops_layer_norm_workspace(1 << 24, 4100, 1) == 0
    assert lib.atlas_ops_layer_norm_workspace((1 << 24) - 1, 4100, 1) > 0
    for width, type_ in ((4100, 0), (8200, 1)):  # a workgroup for each row
        refused(lib.atlas_ops_layer_norm(rows, 1 << 24, width, type_, None, None, 0, 1e-5, p, None, None, None, address, 256), "rows")
        refused(lib.atlas_ops_layer_norm_backward(rows, rows, 1 << 24, width, type_, None, 0, p, p, p, p, p, p, None, address,
                                                  256), "rows")
    refused(lib.atlas_ops_layer_norm_backward(rows, rows, 1 << 24, 4100, 1, None, 0, p, p, p, p, p, p, None, address, 256), "rows")

    for sizes in ((1, 17000, 17000), (1, 1 << 21, 4), (1, 4, 1 << 21), (70000, 4, 4)):
        assert lib.atlas_ops_orthogonalize_workspace(*sizes) == 0
        packed = ops._ORTHOGONAL.pack(p, *sizes, 16, 4, 0, p, 0, 0, 0, 1, 5, 0.9, 1e-7, 1.0, 0.1, 3.0, -4.0, 2.0)
        refused(lib.atlas_ops_orthogonalize(packed, None, None, address, 256), "16384" if sizes[1] == 17000 else "batch")
    assert lib.atlas_ops_orthogonalize_workspace(1, 16384, 1 << 20) > 0


def test_the_abi_refuses_coefficients_beyond_the_planes():
    lib = ops.library()
    err = ctypes.create_string_buffer(256)
    for steps, coefficients in ((3, (30.0, 0.0, 0.0)), (2, (5000.0, 0.0, 0.0)), (1, (1.0, 2500.0, 2000.0)), (9, (-2.0, -1.0, 0.0)),
                                (5, (float("nan"), 0.0, 0.0)), (5, (1.0, 0.0, float("-inf")))):
        packed = ops._ORTHOGONAL.pack(4096, 1, 4, 4, 16, 4, 0, 4096, 0, 0, 0, 1, steps, 0.9, 1e-7, 1.0, 0.1, *coefficients)
        rc = lib.atlas_ops_orthogonalize(packed, 4096, None, ctypes.addressof(err), 256)  # the address is never read
        assert rc == 7 and b"coefficients" in err.value, (steps, coefficients, err.value)


def test_a_decay_gradient_taken_too_early_is_caught(monkeypatch):
    """The gradient of log_decay taken before the correction's own share has left the state's gradient: both the
    comparison with autograd and that with differences have to see it."""
    right = """                D = D - np.outer(kt, de)
                g["log_decay"][b, t, h] = (D * faded).sum()
"""
    wrong = "".join(reversed(right.splitlines(keepends=True)))
    source = inspect.getsource(oo.delta_rule_backward)
    assert source.count(right) == 1
    planted = {}
    exec(source.replace(right, wrong), vars(oo), planted)
    monkeypatch.setattr(oo, "delta_rule_backward", planted["delta_rule_backward"])
    with pytest.raises(AssertionError, match="log_decay"):
        test_delta_reference_matches_autograd()
    with pytest.raises(AssertionError, match="log_decay"):
        test_delta_reference_matches_differences(None)
