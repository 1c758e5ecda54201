"""The gated delta rule on the GPU against the float64 reference, token by token (oracle/ops_oracle.py).

Tolerances.  A chunk's results are chains of about ten float32 products over at most 128 terms; keys of unit
length and rates below one make every step a contraction, so errors add but do not grow: ten sums of 200
terms at sqrt(200) 2^-24 each are 8e-6 of the largest term.  out and the state are held to 2e-5 of the largest
value, gradients, which chain twice as many products, to 4e-5; dlog_decay sums up to 64 differences of such
terms and is held to 1e-4.  bfloat16 results: an ulp, 2^-8, on top.
"""
import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INPUTS = ("q", "k", "v", "log_decay", "beta", "state")


def numpy(t):
    return None if t is None else t.double().cpu().numpy()


def make(B, T, H, Hv, dk, dv, dtype=F32, seed=0, state=True, gates=F32, decay=True):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k = (normal(B, T, H, dk) + 0.3 for _ in range(2))
    q, k = (a / a.norm(dim=-1, keepdim=True).clamp_min(1e-6) for a in (q, k))
    case = dict(q=q.to(dtype), k=k.to(dtype), v=normal(B, T, Hv, dv).to(dtype),
                log_decay=-torch.exp(normal(B, T, Hv) * 1.5 - 3).to(gates) if decay else None,
                beta=torch.sigmoid(normal(B, T, Hv)).to(gates), state=normal(B, Hv, dk, dv) if state else None)
    return {n: None if t is None else t.cuda() for n, t in case.items()}


def close(got, want, tol, what):
    error = np.abs(numpy(got) - want)
    bound = tol * (np.abs(want).max(initial=0.0) + 1e-6) + (2.0 ** -8 * np.abs(want) if got.dtype == BF16 else 0.0)
    assert (error <= bound).all(), (what, float((error / bound).max()))


def check(case, lengths=None, scale=None, seed=9, train=True):
    device_lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    args = [case[n] for n in INPUTS]
    host = [numpy(a) for a in args]
    out, final = ops.delta_rule(*args, lengths=device_lengths, scale=scale)
    want, state, _ = oo.delta_rule(*host, lengths=lengths, scale=scale)
    assert out.dtype == case["v"].dtype and final.dtype == F32 and out.is_contiguous()
    close(out, want, 2e-5, "out")
    close(final, state, 2e-5, "state")
    if not train:
        return
    g = torch.Generator().manual_seed(seed)
    go = torch.randn(out.shape, generator=g).to(out.dtype).cuda()
    gs = torch.randn(final.shape, generator=g).cuda()
    taped, taped_state, tape = ops.delta_rule(*args, lengths=device_lengths, scale=scale, tape=True)
    close(taped, want, 2e-5, "out with a tape")
    close(taped_state, state, 2e-5, "state with a tape")
    grads = ops.delta_rule_backward(go, gs, tape)
    expected = oo.delta_rule_backward(numpy(go), numpy(gs), *host, lengths=lengths, scale=scale)
    for name in INPUTS:
        if case[name] is None:
            assert grads[name] is None
            continue
        assert grads[name].dtype == case[name].dtype and grads[name].shape == case[name].shape
        close(grads[name], expected[name], 1e-4 if name == "log_decay" else 4e-5, "gradient of " + name)
    again = ops.delta_rule_backward(go, gs, tape)
    assert all(grads[n] is None or torch.equal(grads[n], again[n]) for n in INPUTS), "the same bits on every run"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("time", [1, 2, 15, 16, 17, 63, 64, 65, 129, 200])
def test_lengths_around_a_chunk(time, dtype):
    print(f"case: delta rule time {time} {dtype}", flush=True)
    check(make(2, time, 2, 2, 32, 24, dtype, seed=time))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("key,value", [(1, 1), (3, 130), (16, 16), (40, 17), (63, 64), (64, 65), (65, 63), (96, 32),
                                       (127, 20), (128, 128), (128, 1)])
def test_widths(key, value, dtype):
    print(f"case: delta rule widths {key} {value} {dtype}", flush=True)
    check(make(1, 70, 1, 2, key, value, dtype, seed=key + value))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,value_heads", [(1, 1), (1, 4), (2, 6), (3, 3)])
def test_shared_heads(heads, value_heads, dtype):
    print(f"case: delta rule heads {heads} {value_heads} {dtype}", flush=True)
    check(make(2, 100, heads, value_heads, 24, 20, dtype, seed=heads))


@pytest.mark.parametrize("state,decay,gates", [(False, True, F32), (True, False, F32), (True, True, BF16), (False, False, BF16)])
def test_optional_inputs(state, decay, gates):
    print(f"case: delta rule options {state} {decay} {gates}", flush=True)
    check(make(2, 90, 2, 2, 32, 32, BF16, seed=5, state=state, gates=gates, decay=decay), scale=0.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[0, 150], [150, 1], [64, 63], [0, 0], [200, -3], [65, 128]])
def test_ragged_lengths(lengths, dtype):
    """Beyond its length a sequence's inputs are not looked at: they hold NaN and infinities here."""
    print(f"case: delta rule lengths {lengths} {dtype}", flush=True)
    case = make(2, 150, 1, 2, 32, 40, dtype, seed=11)
    valid = [min(150, max(0, n)) for n in lengths]
    for n in ("q", "k", "v", "log_decay", "beta"):
        for b, end in enumerate(valid):
            case[n][b, end:] = float("nan") if n != "v" else float("inf")
    out = ops.delta_rule(*(case[n] for n in INPUTS), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))[0]
    for b, end in enumerate(valid):
        assert (out[b, end:] == 0).all()
    check(case, lengths)
    check({**case, **{n: case[n][:, :12] for n in ("q", "k", "v", "log_decay", "beta")}}, [min(12, n) for n in lengths])


def test_ragged_gradients_of_unused_tokens_are_zero():
    print("case: delta rule unused gradients", flush=True)
    case = make(2, 140, 2, 2, 20, 20)
    lengths = torch.tensor([3, 100], dtype=torch.int32, device="cuda")
    out, final, tape = ops.delta_rule(*(case[n] for n in INPUTS), lengths=lengths, tape=True)
    go = torch.full_like(out, float("nan"))
    go[0, :3], go[1, :100] = 1.0, 1.0
    grads = ops.delta_rule_backward(go, None, tape)
    for n in INPUTS[:-1]:
        assert torch.isfinite(grads[n]).all() and (grads[n][0, 3:] == 0).all() and (grads[n][1, 100:] == 0).all(), n


def test_hard_keys():
    """The same key at every token with rate one (the inverse's largest entries), 0/1 keys as spikes with a
    small rate, rates of zero, keys of zero, and rates up to two."""
    print("case: delta rule hard keys", flush=True)
    case = make(1, 150, 1, 1, 32, 32, seed=3)
    case["k"][:] = case["k"][:, :1]
    case["beta"][:] = 1.0
    check(case)
    case["log_decay"][:] = 0.0
    check(case)
    case = make(1, 150, 1, 1, 32, 32, seed=4)
    case["k"] = (case["k"] > 0.2).float()
    case["beta"] *= 0.05
    check(case)
    case = make(1, 150, 1, 1, 32, 32, seed=5)
    case["beta"][:, ::2] = 0.0
    case["k"][:, 5:80:3] = 0.0
    check(case)
    case["beta"] = 2.0 * case["beta"]
    check(case)


def test_decays_of_every_size():
    """-inf, the type's lowest value and large decays empty the state; small ones between them keep their
    accuracy, as the running sums are differences of 64-bit numbers."""
    print("case: delta rule decays", flush=True)
    case = make(2, 140, 1, 2, 24, 24, seed=6)
    case["log_decay"][0, 10::31] = -float("inf")
    case["log_decay"][1, 7::17] = torch.finfo(F32).min
    case["log_decay"][1, 9::13] = -40.0
    check(case)
    case["log_decay"] = case["log_decay"].bfloat16()
    check(case)
    emptied = make(1, 70, 1, 1, 16, 16, seed=7)
    emptied["log_decay"][0, 66] = -float("inf")
    whole, state = ops.delta_rule(*(emptied[n] for n in INPUTS))
    late = {n: None if n == "state" else emptied[n][:, 66:] for n in INPUTS}
    tail, tail_state = ops.delta_rule(*(late[n] for n in INPUTS))
    close(whole[:, 66:], numpy(tail), 2e-5, "after the state was emptied")
    close(state, numpy(tail_state), 2e-5, "state")


def test_a_nan_stays_in_its_head():
    print("case: delta rule NaN", flush=True)
    for name, at in (("v", (0, 3, 1, 2)), ("log_decay", (0, 3, 1)), ("beta", (0, 3, 1))):
        case = make(2, 80, 2, 2, 16, 16, seed=8)
        case[name][at] = float("nan")
        for tokens in (80, 10):
            part = [case[n] if n == "state" else case[n][:, :tokens] for n in INPUTS]
            out, state = ops.delta_rule(*part)
            assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :, 0]).all() and torch.isfinite(out[0, :3]).all()
            assert torch.isnan(out[0, 4:, 1]).any() and torch.isnan(state[0, 1]).any()
            assert torch.isfinite(state[1]).all() and torch.isfinite(state[0, 0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    print(f"case: delta rule strides {dtype}", flush=True)
    case = make(3, 80, 2, 2, 20, 12, dtype, seed=10)
    args = [case[n] for n in INPUTS]
    want = ops.delta_rule(*args, tape=True)
    g = torch.Generator().manual_seed(1)
    go = torch.randn(want[0].shape, generator=g).to(dtype).cuda()
    grads = ops.delta_rule_backward(go, None, want[2])
    # tick-major memory, heads outside, odd starts, and a last axis that is not contiguous
    moved = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in args[:5]]
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in args[:5]]
    padded = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in args[:5]]
    turned = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in args[:5]]
    for inputs in (moved, heads, padded, turned):
        state = args[5].transpose(2, 3).contiguous().transpose(2, 3)
        out, final, tape = ops.delta_rule(*inputs, state, tape=True)
        assert torch.equal(out, want[0]) and torch.equal(final, want[1])
        for grad_out in (go, go.transpose(0, 1).contiguous().transpose(0, 1), go.transpose(2, 3).contiguous().transpose(2, 3)):
            got = ops.delta_rule_backward(grad_out, None, tape)
            assert all(torch.equal(got[n], grads[n]) for n in INPUTS)
    # one q and k for the whole batch, a gradient of a sum
    shared = [t[:1].expand_as(t) for t in args[:2]]
    a = ops.delta_rule(*shared, *args[2:], tape=True)
    b = ops.delta_rule(*(t.contiguous() for t in shared), *args[2:], tape=True)
    assert torch.equal(a[0], b[0])
    ones = torch.ones((), dtype=dtype, device="cuda").expand(want[0].shape)
    ga, gb = ops.delta_rule_backward(ones, None, a[2]), ops.delta_rule_backward(ones.contiguous(), None, b[2])
    assert all(torch.equal(ga[n], gb[n]) for n in INPUTS)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("key,value,heads,value_heads", [(1, 1, 1, 1), (33, 17, 2, 4), (128, 128, 2, 2), (100, 66, 1, 3)])
def test_steps_equal_the_sequence(key, value, heads, value_heads, dtype):
    print(f"case: delta rule steps {key} {value} {dtype}", flush=True)
    case = make(3, 20, heads, value_heads, key, value, dtype, seed=12)
    args = [case[n] for n in INPUTS]
    want, final, _ = oo.delta_rule(*(numpy(a) for a in args))
    state = args[5].clone()
    version = state._version
    for t in range(20):
        out = ops.delta_rule_step(*(a[:, t] for a in args[:5]), state)
        close(out, want[:, t], 2e-5, f"out at {t}")
    assert state._version == version + 20
    close(state, final, 2e-5, "state")


def test_segments_equal_the_whole():
    print("case: delta rule segments", flush=True)
    case = make(2, 300, 2, 2, 48, 48, seed=13)
    args = [case[n] for n in INPUTS]
    whole, final = ops.delta_rule(*args)
    state, parts, at = args[5], [], 0
    for size in (130, 1, 15, 17, 64, 73):
        out, state = ops.delta_rule(*(a[:, at:at + size] for a in args[:5]), state)
        parts.append(out)
        at += size
    assert at == 300
    close(torch.cat(parts, dim=1), numpy(whole), 2e-5, "out")
    close(state, numpy(final), 2e-5, "state")


def test_gradients_match_differences():
    print("case: delta rule differences", flush=True)
    case = make(1, 130, 1, 2, 12, 10, seed=14)
    args = [case[n] for n in INPUTS]
    g = torch.Generator().manual_seed(2)
    go, gs = torch.randn(1, 130, 2, 10, generator=g).cuda(), torch.randn(1, 2, 12, 10, generator=g).cuda()
    grads = ops.delta_rule_backward(go, gs, ops.delta_rule(*args, tape=True)[2])
    for i, name in enumerate(INPUTS):
        direction = torch.randn(args[i].shape, generator=g).cuda()
        values = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * 2e-3 * direction
            out, final = ops.delta_rule(*moved)
            values.append(float((out.double() * go).sum() + (final.double() * gs).sum()))
        difference, slope = (values[0] - values[1]) / 4e-3, float((grads[name].double() * direction).sum())
        # float32 results of order 1 summed over 1300 values leave 1e-5 / 4e-3 = 3e-3, curvature 4e-6 of its size
        assert abs(difference - slope) <= 0.02 + 2e-3 * abs(slope), (name, difference, slope)


def test_empty():
    print("case: delta rule empty", flush=True)
    case = make(2, 5, 1, 1, 8, 8)
    args = [case[n] for n in INPUTS]
    none = [a[:, :0] for a in args[:5]]
    out, final, tape = ops.delta_rule(*none, args[5], tape=True)
    assert out.shape == (2, 0, 1, 8) and torch.equal(final, args[5]) and final.data_ptr() != args[5].data_ptr()
    gs = torch.randn_like(final)
    grads = ops.delta_rule_backward(out, gs, tape)
    assert torch.equal(grads["state"], gs) and grads["q"].shape == (2, 0, 1, 8)
    out, final = ops.delta_rule(*none)
    assert (final == 0).all() and final.shape == (2, 1, 8, 8)
    nobody = [a[:0] for a in args]
    out, final = ops.delta_rule(*nobody)
    assert out.shape == (0, 5, 1, 8) and final.shape == (0, 1, 8, 8)
    assert ops.delta_rule_step(*(a[:0, 0] for a in args[:5]), args[5][:0]).shape == (0, 1, 8)


def test_refusals():
    print("case: delta rule refusals", flush=True)
    case = make(2, 5, 2, 4, 8, 8)
    q, k, v, g, b, s = (case[n] for n in INPUTS)
    lengths = torch.tensor([1, 2], device="cuda")
    for call in (lambda: ops.delta_rule(q, k[:, :4], v, g, b), lambda: ops.delta_rule(q, k, v[:, :4], g, b),
                 lambda: ops.delta_rule(q, k, v[:, :, :3], g[..., :3], b[..., :3]),
                 lambda: ops.delta_rule(q, k, v, g[..., :2], b), lambda: ops.delta_rule(q, k, v, g, b[:1]),
                 lambda: ops.delta_rule(q, k.bfloat16(), v, g, b), lambda: ops.delta_rule(q, k, v.bfloat16(), g, b),
                 lambda: ops.delta_rule(q.half(), k.half(), v.half(), g, b), lambda: ops.delta_rule(q, k, v, g.double(), b),
                 lambda: ops.delta_rule(q, k, v, g, b, s.bfloat16()), lambda: ops.delta_rule(q, k, v, g, b, s[:, :2]),
                 lambda: ops.delta_rule(q, k, v, g, b, lengths=lengths),
                 lambda: ops.delta_rule(q, k, v, g, b, lengths=lengths.int()[:1]),
                 lambda: ops.delta_rule(q[0], k[0], v[0], g[0], b[0]), lambda: ops.delta_rule(q, k, v, g, None),
                 lambda: ops.delta_rule(q, k, v.clone().requires_grad_(), g, b),
                 lambda: ops.delta_rule(torch.zeros(1, 1, 1, 129, device="cuda"), torch.zeros(1, 1, 1, 129, device="cuda"),
                                        v[:1, :1, :1], g[:1, :1, :1], b[:1, :1, :1]),
                 lambda: ops.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], b[:, 0], None),
                 lambda: ops.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], b[:, 0], s.transpose(2, 3)),
                 lambda: ops.delta_rule_step(q, k, v, g, b, s)):
        with pytest.raises(ValueError):
            call()
    out, final, tape = ops.delta_rule(q, k, v, g, b, tape=True)
    for call in (lambda: ops.delta_rule_backward(out[:1], None, tape), lambda: ops.delta_rule_backward(out.bfloat16(), None, tape),
                 lambda: ops.delta_rule_backward(out, final[:1], tape), lambda: ops.delta_rule_backward(out, final.half(), tape)):
        with pytest.raises(ValueError):
            call()


def test_offsets_beyond_32_bits():
    """Batches and ticks more than 2^31 elements apart."""
    print("case: delta rule offsets", flush=True)
    case = make(2, 70, 1, 1, 16, 16, BF16, seed=15)
    args = [case[n] for n in INPUTS]
    want = ops.delta_rule(*args, tape=True)
    go = torch.ones_like(want[0])
    grads = ops.delta_rule_backward(go, None, want[2])
    memory = torch.empty((1 << 31) + 5000, dtype=BF16, device="cuda")
    for i in range(3):
        far = memory.as_strided((2, 70, 1, 16), ((1 << 31), 16, 16, 1))
        far.copy_(args[i])
        inputs = list(args)
        inputs[i] = far
        out, final, tape = ops.delta_rule(*inputs, tape=True)
        assert torch.equal(out, want[0]) and torch.equal(final, want[1])
        got = ops.delta_rule_backward(go, None, tape)
        assert all(torch.equal(got[n], grads[n]) for n in INPUTS)


def test_backward_on_another_stream():
    print("case: delta rule streams", flush=True)
    case = make(2, 200, 2, 2, 32, 32, seed=16)
    args = [case[n] for n in INPUTS]
    out, final, tape = ops.delta_rule(*args, tape=True)
    go = torch.ones_like(out)
    want = ops.delta_rule_backward(go, None, tape)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.delta_rule_backward(go, None, tape)
    del tape
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(got[n], want[n]) for n in INPUTS)


@pytest.mark.parametrize("key", [64, 128])
def test_bfloat16_outputs_are_rounded_once(key):
    """A bfloat16 result that is a float32 one rounded once lands beside the exact result's rounding only where
    that lies within the float32 error of the middle between two bfloat16 values.  Errors of the four chained sums
    (K S, T R, Q S, P E), each of some twelve roundings of 2^-25, come to 2e-7 of the results' size, 5e-7 at most.  An
    error of r puts 0.8 r 2^7.5 E[1 / |x|] of normally distributed x on the other side, with E[1 / |x|] = 7 (cut
    where a spacing is the error): 5e-4 of the values at 5e-7.  Held to twice that; operands of 16 bits give 3e-3."""
    print(f"case: delta rule rounding {key}", flush=True)
    case = make(1, 300, 2, 2, key, 128, BF16, seed=key)
    args = [case[n] for n in INPUTS]
    want = torch.from_numpy(oo.delta_rule(*(numpy(a) for a in args))[0]).to(BF16).cuda()
    for tape in (False, True):
        other = (ops.delta_rule(*args, tape=tape)[0] != want).double().mean()
        assert other <= 1e-3, float(other)


def same(a, b):
    """The same values, NaN where NaN is."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("key,time", [(24, 12), (24, 150), (64, 150), (100, 150), (100, 330)])
def test_unused_tokens_leave_any_state_as_it_is(key, time, dtype):
    """NaN and infinities in the state of a sequence without tokens, or that its last token left there, stay where
    they are; backwards the same for the final state's gradient."""
    print(f"case: delta rule unused {key} {time} {dtype}", flush=True)
    case = make(3, time, 1, 2, key, 40, dtype, seed=17)
    case["state"][0, 0, 3, 5], case["state"][0, 1, 1, 0] = float("nan"), float("inf")
    case["v"][1, min(time, 64) - 1, 1, 7] = float("inf")
    lengths = [0, min(time, 64), time]
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    args = [case[n] for n in INPUTS]
    for tape in (False, True):
        out, final = ops.delta_rule(*args, lengths=device_lengths, tape=tape)[:2]
        assert same(final[0], args[5][0]) and (out[0] == 0).all()
        alone, left = ops.delta_rule(*(a[1:2] if a is args[5] else a[1:2, :lengths[1]] for a in args), tape=True)[:2]
        if tape:  # without one, short sequences take another kernel
            assert same(final[1], left[0]) and same(out[1, :lengths[1]], alone[0]) and (out[1, lengths[1]:] == 0).all()
        assert torch.isfinite(final[2]).all()
    case["v"][1, min(time, 64) - 1, 1, 7] = 1.0
    case["state"][0] = 1.0
    out, _, tape = ops.delta_rule(*args, lengths=device_lengths, tape=True)
    go, gs = torch.ones_like(out), torch.ones_like(args[5])
    want = ops.delta_rule_backward(go, gs, tape)
    gs[0, 0, 3, 5], gs[0, 1, 1, 0] = float("nan"), float("inf")
    grads = ops.delta_rule_backward(go, gs, tape)
    assert same(grads["state"][0], gs[0])
    for n in INPUTS[:5]:
        assert (grads[n][0] == 0).all() and (grads[n][1, lengths[1]:] == 0).all() and torch.equal(grads[n], want[n]), n


def test_sizes_beyond_the_limits_are_invalid_arguments():
    print("case: delta rule limits", flush=True)
    one = torch.ones(1, device="cuda")
    q, v, gate = one.expand(65536, 13, 1, 1), one.expand(65536, 13, 1, 1), one.expand(65536, 13, 1)
    with pytest.raises(ValueError, match="65535"):
        ops.delta_rule(q, q, v, gate, gate)
    with pytest.raises(ValueError, match="65535"):
        ops.delta_rule_step(q[:, 0], q[:, 0], v[:, 0], gate[:, 0], gate[:, 0], torch.ones(65536, 1, 1, 1, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("key,value,heads,value_heads,time,lengths", [
    (128, 128, 1, 1, 129, None), (128, 128, 1, 2, 192, None), (128, 40, 2, 2, 200, [200, 65]), (128, 128, 1, 3, 300, [300, 190]),
    (128, 17, 1, 1, 321, None), (96, 40, 1, 2, 129, [128, 129]), (96, 40, 2, 2, 192, None), (96, 72, 1, 2, 256, [64, 256]),
    (96, 40, 1, 1, 300, None), (65, 33, 1, 4, 385, [385, 0])])
def test_wide_keys_over_many_chunks(key, value, heads, value_heads, time, lengths, dtype):
    """Odd and even numbers of chunks, from three on, of the kernels for keys above 64."""
    print(f"case: delta rule wide {key} {value} {heads} {value_heads} {time} {lengths} {dtype}", flush=True)
    check(make(2, time, heads, value_heads, key, value, dtype, seed=key + time), lengths)


def test_a_faulty_key_or_query_stays_behind_its_token():
    """A query's fault reaches its own output alone, a key's its own and later tokens of its head."""
    print("case: delta rule faulty keys", flush=True)
    for fault in (float("nan"), float("inf")):
        for tokens in (150, 10):
            case = make(2, 150, 2, 4, 24, 40, seed=18)
            case["q"][0, 5, 1, 2] = fault
            case["k"][1, 5, 0, 3] = fault
            out, state = ops.delta_rule(*(case[n] if n == "state" else case[n][:, :tokens] for n in INPUTS))
            assert not torch.isfinite(out[0, 5, 2:]).any() and torch.isfinite(out[0, 5, :2]).all()
            out[0, 5] = 0.0
            assert torch.isfinite(out[0]).all() and torch.isfinite(state[0]).all()
            assert torch.isfinite(out[1, :5]).all() and torch.isfinite(out[1, :, 2:]).all() and torch.isfinite(state[1, 2:]).all()
            assert not torch.isfinite(out[1, 6:, :2]).any() and not torch.isfinite(state[1, :2]).all(dim=-2).any()
