"""Linear attention on the GPU against the float64 reference (oracle/ops_oracle.py).

Tolerances, in roundings of 2^-24 of M, the same quantity with every input replaced by its magnitude, which bounds the sum of
the magnitudes of its terms.  Operands are held to 24 bits and products taken to 2^-23; decays are within 2^-22; a result
adds at most 128 / 32 + 64 / 32 blocks of up to six products one after the other, and a state at most 14 roundings for each chunk
of 32 or 64 tokens that it passes and one for each segment (at most 64 chunks apart, far fewer than chunks): UNITS(T) = 64 + 16 T / 32.
The gradient of a decay is a sum of q . dQ and k . dK over the tokens from there on: its M adds those of the tokens behind.
A bfloat16 result is rounded once (2^-8 of its value).
"""
import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ULP = 2.0 ** -24
ROUND = {F32: 0.0, BF16: 2.0 ** -8}


def numpy(t):
    return None if t is None else t.double().cpu().numpy()


def make(B, T, H, Hv, dk, dv, dtype=F32, decay="token", state=True, seed=0, decay_type=F32):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, v = normal(B, T, H, dk), normal(B, T, H, dk) / dk ** 0.5, normal(B, T, Hv, dv)
    decays = None if decay is None else -torch.exp(-6.0 + 6.0 * torch.rand(*((Hv,) if decay == "head" else (B, T, Hv)), generator=g))
    start = normal(B, Hv, dk, dv) if state else None
    case = dict(q=q.to(dtype), k=k.to(dtype), v=v.to(dtype), log_decay=None if decays is None else decays.to(decay_type), state=start)
    return {n: None if t is None else t.cuda() for n, t in case.items()}


def magnitudes(case):
    return {n: None if a is None else a if n == "log_decay" else np.abs(a) for n, a in case.items()}


def close(got, want, size, units, what):
    bound = units * ULP * size + ROUND.get(got.dtype, 0.0) * np.abs(want) + 1e-37
    error = np.abs(numpy(got) - want)
    assert np.isfinite(numpy(got)).all() and (error <= bound).all(), (what, float((error / bound).max()))


def check(case, lengths=None, scale=None, grad_state=True, train=True):
    a = {n: numpy(t) for n, t in case.items()}
    T, on = a["q"].shape[1], None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    units = 64 + T / 2
    out, final = ops.linear_attention(**case, lengths=on, scale=scale)
    want, last, _ = oo.linear_attention(**a, lengths=lengths, scale=scale)
    size, size_last, _ = oo.linear_attention(**magnitudes(a), lengths=lengths, scale=None if scale is None else abs(scale))
    assert out.dtype == case["v"].dtype and out.is_contiguous()
    close(out, want, size, units, "out")
    close(final, last, size_last, units, "state")
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert (out[b, max(0, n):] == 0).all()
    if not train:
        return out, final
    g = torch.Generator().manual_seed(99)
    go = torch.randn(out.shape, generator=g).to(out.dtype).cuda()
    gs = torch.randn(final.shape, generator=g).cuda() if grad_state else None
    out2, final2, tape = ops.linear_attention(**case, lengths=on, scale=scale, tape=True)
    close(out2, want, size, units, "out with a tape")
    close(final2, last, size_last, units, "state with a tape")
    final2.zero_()   # the caller's own from here on
    grads = ops.linear_attention_backward(go, gs, tape)
    wanted = oo.linear_attention_backward(numpy(go), numpy(gs), **a, lengths=lengths, scale=scale)
    m, mgo, mgs = magnitudes(a), np.abs(numpy(go)), None if gs is None else np.abs(numpy(gs))
    sizes = oo.linear_attention_backward(mgo, mgs, **m, lengths=lengths, scale=None if scale is None else abs(scale))
    group = a["v"].shape[2] // a["q"].shape[2]
    for name, got in grads.items():
        assert (got is None) == (case[name] is None)
        if got is None:
            continue
        assert got.shape == case[name].shape and got.dtype == case[name].dtype, name
        size = sizes[name]
        if name == "log_decay":
            per_head = dict(m, q=np.repeat(m["q"], group, 2), k=np.repeat(m["k"], group, 2))
            each = oo.linear_attention_backward(mgo, mgs, **per_head, lengths=lengths, scale=None if scale is None else abs(scale))
            terms = (per_head["q"] * each["q"]).sum(-1) + (per_head["k"] * each["k"]).sum(-1)
            size = np.cumsum(terms[:, ::-1], axis=1)[:, ::-1] + (0.0 if gs is None else (mgs * size_last).sum(axis=(2, 3))[:, None])
            size = size.sum(axis=(0, 1)) if size.shape[2:] == got.shape and got.dim() == 1 else size
        close(got, wanted[name], size, units, name)
    again = ops.linear_attention_backward(go, gs, tape)
    assert all(x is None if y is None else torch.equal(x, y) for x, y in zip(grads.values(), again.values())), "the same bits on every run"
    return out, final


# lengths around a token, a step, chunks of 32 and 64 and several segments; widths on both sides of 64, 32 and 4, odd ones
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,Hv,dk,dv", [(1, 1, 1, 1, 1, 1), (2, 2, 1, 2, 3, 5), (1, 12, 2, 2, 16, 16), (1, 13, 2, 2, 16, 24), (2, 31, 1, 1, 64, 64),
                                            (1, 32, 1, 3, 65, 64), (1, 33, 2, 2, 64, 65), (2, 63, 1, 1, 128, 128), (1, 64, 1, 2, 33, 127), (3, 65, 2, 4, 40, 72),
                                            (1, 100, 4, 4, 64, 64), (1, 127, 1, 1, 96, 128), (2, 128, 1, 2, 128, 32), (1, 129, 1, 1, 17, 100),
                                            (1, 200, 1, 1, 128, 128), (1, 300, 1, 4, 72, 48), (1, 1000, 1, 2, 24, 16)])
def test_matches_the_reference(B, T, H, Hv, dk, dv, dtype):
    print(f"case: linear attention {B} x {T}, {H} and {Hv} heads of {dk} x {dv} {dtype}", flush=True)
    check(make(B, T, H, Hv, dk, dv, dtype))
    check(make(B, T, H, Hv, dk, dv, dtype, decay="head", state=False), grad_state=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_segment(dtype):
    """So many heads that a sequence is not split."""
    print(f"case: linear attention one segment {dtype}", flush=True)
    check(make(33, 150, 8, 16, 16, 20, dtype))
    check(make(33, 150, 16, 16, 16, 20, dtype, decay="head"), lengths=[150, 0, 1] + [7 * i % 151 for i in range(30)])


@pytest.mark.parametrize("dtype,T", [(F32, 650), (BF16, 1290)])
@pytest.mark.parametrize("dk,dv", [(20, 24), (68, 12)])
def test_segments_of_several_chunks(dk, dv, dtype, T):
    """Segments of three chunks each, which end between the places where a decay's gradient starts anew; widths that one kernel
    holds both ways round and widths that take two."""
    print(f"case: linear attention segments {T} tokens {dk} x {dv} {dtype}", flush=True)
    check(make(9, T, 4, 8, dk, dv, dtype), lengths=[T, 0, 1, T - 1, T // 2, 192, 193, 40, T // 3])
    check(make(9, T, 8, 8, dk, dv, dtype, decay="head", state=False), grad_state=False)


@pytest.mark.parametrize("decay", [None, "token", "head"])
@pytest.mark.parametrize("lengths", [[70, 33, 0], [1, 64, 200], [200, 199, -3], [65, 300, 32]])
def test_lengths(lengths, decay):
    print(f"case: linear attention lengths {lengths} {decay}", flush=True)
    for dtype in (F32, BF16):
        case = make(3, 200, 1, 2, 40, 48, dtype, decay=decay)
        for name in ("q", "k", "v"):   # what lies behind a sequence's end is not looked at
            for b, n in enumerate(lengths):
                case[name][b, max(0, n):] = 0.0
        out, final = check(case, [min(200, max(0, n)) for n in lengths])
        dirty = {n: None if t is None else t.clone() for n, t in case.items()}
        for name in ("q", "k", "v", "log_decay"):
            if dirty[name] is not None and dirty[name].dim() > 1:
                for b, n in enumerate(lengths):
                    dirty[name][b, max(0, n):] = float("nan")
        on = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        go = torch.ones_like(out)
        results = []
        for c in (case, dirty):
            o, f, tape = ops.linear_attention(**c, lengths=on, tape=True)
            grad = go.clone()
            if c is dirty:
                for b, n in enumerate(lengths):
                    grad[b, max(0, n):] = float("nan")
            results.append([o, f, *(g for g in ops.linear_attention_backward(grad, f * 0 + 1, tape).values() if g is not None)])
        assert all(torch.equal(x, y) for x, y in zip(*results))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays_of_every_kind(dtype):
    print(f"case: linear attention decays {dtype}", flush=True)
    check(make(2, 150, 1, 2, 32, 32, dtype, decay=None))
    check(make(2, 150, 1, 2, 32, 32, dtype, decay_type=BF16))
    check(make(2, 150, 1, 2, 32, 32, dtype, decay="head", decay_type=BF16), scale=-0.3)
    case = make(2, 150, 1, 2, 32, 32, dtype)
    case["log_decay"] *= 40.0                       # forgets within a tick
    check(case)
    case["log_decay"][:, ::7] = 0.0
    check(case)
    case["log_decay"][:, 60] = -float("inf")        # empties the state; the reference's exponential is zero as well
    check(case)
    case = make(1, 140, 1, 1, 16, 16, dtype)
    case["log_decay"] = -0.02 * case["log_decay"]   # grows
    check(case)


def test_long_sums_of_decays():
    """Small decays after large ones: sums of log decays in 32 bits would lose them."""
    print("case: linear attention long sums", flush=True)
    case = make(1, 2000, 1, 1, 16, 16)
    case["log_decay"][:, ::64] = -90.0
    case["log_decay"][:, 1::64] = -1e-5
    check(case)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    print(f"case: linear attention strides {dtype}", flush=True)
    B, T, H, d = 2, 70, 2, 24
    g = torch.Generator().manual_seed(5)
    packed = torch.randn(B, T, 3, H, d, generator=g).to(dtype).cuda()
    gates = -torch.rand(B, H, T, generator=g).cuda()
    q, k, v = packed.unbind(2)
    check(dict(q=q, k=k, v=v, log_decay=gates.transpose(1, 2), state=None))
    heads_first = torch.randn(3, B, H, T, d, generator=g).to(dtype).cuda().transpose(2, 3)
    check(dict(q=heads_first[0], k=heads_first[1], v=heads_first[2], log_decay=gates[:, :, :1].transpose(1, 2).expand(B, T, H), state=None))
    # off 16 bytes, a last axis that is not contiguous, broadcast over the batch, decays of every second head
    flat = torch.randn(B * T * H * d + 1, generator=g).to(dtype).cuda()[1:].view(B, T, H, d)
    turned = torch.randn(B, T, d, H, generator=g).to(dtype).cuda().transpose(2, 3)
    check(dict(q=flat, k=turned, v=flat[:1].expand(B, T, H, d), log_decay=-torch.rand(2 * H, generator=g).cuda()[::2],
               state=torch.randn(B, H, d, d, generator=g).cuda().transpose(2, 3)))


def test_gradients_of_strided_results():
    print("case: linear attention gradient strides", flush=True)
    case = make(2, 70, 2, 2, 24, 40)
    out, final, tape = ops.linear_attention(**case, tape=True)
    go, gs = torch.randn_like(out), torch.randn_like(final)
    want = ops.linear_attention_backward(go, gs, tape)
    strange = torch.empty(2, 2, 70, 80, device="cuda").transpose(1, 2)[..., ::2].copy_(go)
    for grad in (strange, go.transpose(0, 1).contiguous().transpose(0, 1)):
        got = ops.linear_attention_backward(grad, gs.transpose(2, 3).contiguous().transpose(2, 3), tape)
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = ops.linear_attention_backward(go[:1, :1, :1].expand(out.shape), None, tape)
    same = ops.linear_attention_backward(go[:1, :1, :1].expand(out.shape).contiguous(), None, tape)
    assert all(torch.equal(one[n], same[n]) for n in one)


def test_tokens_far_apart():
    """More than 2^24 elements from token to token: the results are those of a contiguous copy, bit by bit."""
    T, far = 18, (1 << 24) + 8
    memory = torch.zeros((T - 1) * far + 64, dtype=BF16, device="cuda")
    spread = memory.as_strided((2, T, 2, 8), (32, far, 8, 1))
    case = make(2, T, 2, 2, 8, 8, BF16)
    gs = torch.randn(2, 2, 8, 8, device="cuda")
    want = ops.linear_attention(**case, tape=True)
    go = torch.randn(want[0].shape, device="cuda").to(BF16)
    grads = ops.linear_attention_backward(go, gs, want[2])
    for name in ("q", "v"):
        spread.copy_(case[name])
        got = ops.linear_attention(**dict(case, **{name: spread}), tape=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    spread.copy_(go)
    again = ops.linear_attention_backward(spread, gs, want[2])
    assert all(torch.equal(again[n], grads[n]) for n in grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_fault_reaches_its_own_and_later_tokens(dtype):
    print(f"case: linear attention faults {dtype}", flush=True)
    case = make(1, 200, 1, 2, 20, 70, dtype)
    clean, _ = ops.linear_attention(**case)
    for name, bad in (("k", float("nan")), ("v", float("inf")), ("v", float("nan")), ("q", float("nan")), ("log_decay", float("nan"))):
        for t in (0, 5, 37, 63, 64, 130, 199):
            dirty = dict(case, **{name: case[name].clone()})
            dirty[name][0, t, 0, ...] = bad
            out, _ = ops.linear_attention(**dirty)
            assert torch.equal(out[:, :t], clean[:, :t]), (name, t)
            assert not torch.isfinite(out[0, t, 0]).any(), (name, t)
            if name == "q":
                assert torch.equal(out[:, t + 1:], clean[:, t + 1:])
            else:
                assert not torch.isfinite(out[0, t:, 0]).any(), (name, t)
    dirty = dict(case, v=case["v"].clone())
    dirty["v"][0, 70, 1, 33] = float("nan")   # one column of one head
    out, final = ops.linear_attention(**dirty)
    bad = ~torch.isfinite(out)
    assert bad[0, 70:, 1, 33].all() and bad.sum() == 130 and torch.equal(out[~bad], clean[~bad])
    assert (~torch.isfinite(final))[0, 1, :, 33].all() and (~torch.isfinite(final)).sum() == 20


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,Hv,dk,dv", [(1, 1, 1, 1, 1), (3, 2, 4, 24, 20), (2, 1, 3, 65, 33), (5, 8, 8, 128, 128), (1, 2, 2, 100, 7), (2, 1, 1, 128, 64)])
def test_steps_continue_a_sequence(B, H, Hv, dk, dv, dtype):
    print(f"case: linear attention steps {B}, {H} and {Hv} heads of {dk} x {dv} {dtype}", flush=True)
    for decay in ("token", "head", None):
        case = make(B, 20, H, Hv, dk, dv, dtype, decay=decay, seed=3)
        a = {n: numpy(t) for n, t in case.items()}
        want, last, _ = oo.linear_attention(**a)
        size, size_last, _ = oo.linear_attention(**magnitudes(a))
        state, outs = case["state"].clone(), []
        for t in range(20):
            gate = case["log_decay"]
            version = state._version
            outs.append(ops.linear_attention_step(case["q"][:, t], case["k"][:, t], case["v"][:, t], gate[:, t] if decay == "token" else gate, state))
            assert state._version > version
        close(torch.stack(outs, 1), want, size, 80, "out")
        close(state, last, size_last, 80, "state")
        most = ops.SHORT_LINEAR
        short = {n: t[:, :most] if n in "qkv" or n == "log_decay" and decay == "token" else t for n, t in case.items()}
        out, final = ops.linear_attention(**short)
        assert torch.equal(out, torch.stack(outs[:most], 1)), "the same kernel"


def test_bfloat16_outputs_round_once():
    """Products of 24 bits: hardly a value rounds to the other neighbour of the exact one."""
    print("case: linear attention rounding", flush=True)
    case = make(1, 1024, 2, 2, 128, 128, BF16)
    out, _ = ops.linear_attention(**case)
    want = torch.from_numpy(oo.linear_attention(**{n: numpy(t) for n, t in case.items()})[0]).to(BF16).cuda()
    assert (out != want).float().mean() < 1e-3


def test_empty():
    print("case: linear attention empty", flush=True)
    for B, T in ((0, 5), (2, 0)):
        case = make(B, T, 1, 2, 8, 4)
        out, final, tape = ops.linear_attention(**case, tape=True)
        assert out.shape == (B, T, 2, 4) and torch.equal(final, case["state"])
        gs = torch.ones_like(final)
        grads = ops.linear_attention_backward(out, gs, tape)
        assert torch.equal(grads["state"], gs) and all(g.shape == case[n].shape for n, g in grads.items())
    case = make(0, 5, 1, 2, 8, 4, decay="head", state=False)
    out, final, tape = ops.linear_attention(**case, tape=True)
    assert final.shape == (0, 2, 8, 4)
    assert (ops.linear_attention_backward(out, None, tape)["log_decay"] == 0).all()
    assert ops.linear_attention_step(*(case[n][:, 0] for n in "qkv"), case["log_decay"], final).shape == (0, 2, 4)


def test_refusals():
    print("case: linear attention refusals", flush=True)
    c = make(2, 5, 2, 4, 8, 4)
    q, k, v, g, s = c["q"], c["k"], c["v"], c["log_decay"], c["state"]
    out, final, tape = ops.linear_attention(q, k, v, g, s, tape=True)
    wide = torch.zeros(2, 5, 2, 129, device="cuda")
    dout, _, dtape = ops.delta_rule(q, k, v, g, -g, tape=True)
    for call in (lambda: ops.linear_attention(q, k[:, :4], v, g), lambda: ops.linear_attention(q, k, v[:, :, :3], g[:, :, :3]),
                 lambda: ops.linear_attention(q, k, v, g[:, :4]), lambda: ops.linear_attention(q, k, v, g[0, 0, :3]), lambda: ops.linear_attention(q, k, v, g[0]),
                 lambda: ops.linear_attention(wide, wide, v, g), lambda: ops.linear_attention(q, k, torch.zeros(2, 5, 4, 129, device="cuda"), g),
                 lambda: ops.linear_attention(q.half(), k.half(), v.half(), g), lambda: ops.linear_attention(q.bfloat16(), k, v, g),
                 lambda: ops.linear_attention(q, k, v, g.half()), lambda: ops.linear_attention(q, k, v, g, s.bfloat16()), lambda: ops.linear_attention(q, k, v, g, s[:1]),
                 lambda: ops.linear_attention(q, k, v, g, lengths=torch.tensor([1, 2], device="cuda")), lambda: ops.linear_attention(q, k, v, g, lengths=[1, 2]),
                 lambda: ops.linear_attention(q[0], k[0], v[0], g[0]), lambda: ops.linear_attention(q, k, v[..., :0], g), lambda: ops.linear_attention(q[:, :, :0], k[:, :, :0], v, g),
                 lambda: ops.linear_attention(q.clone().requires_grad_(), k, v, g), lambda: ops.linear_attention(q, k, v, -0.1), lambda: ops.linear_attention(None, k, v, g),
                 lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], None), lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s.transpose(2, 3)),
                 lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s.transpose(0, 1).contiguous().transpose(0, 1)),
                 lambda: ops.linear_attention_backward(out[:1], None, tape), lambda: ops.linear_attention_backward(out.bfloat16(), None, tape),
                 lambda: ops.linear_attention_backward(out, final[:1], tape), lambda: ops.linear_attention_backward(out, None, None),
                 lambda: ops.linear_attention_backward(dout, None, dtape), lambda: ops.delta_rule_backward(out, None, tape)):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        ops.linear_attention(q.clone().requires_grad_(), k, v, g)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_single_token_of_any_stride(dtype):
    """One token has no distance to the next: (time, batch, ...) turned, whose time stride passes 2^24 elements."""
    print(f"case: linear attention single token {dtype}", flush=True)
    far = lambda t: t.as_strided(t.shape, (t.stride(0), 1 << 25, *t.stride()[2:]))  # noqa: E731
    case = make(2, 1, 2, 2, 8, 8, dtype)
    want = ops.linear_attention(**case, tape=True)
    go, gs = torch.randn(want[0].shape, device="cuda").to(dtype), torch.randn(want[1].shape, device="cuda")
    grads = ops.linear_attention_backward(go, gs, want[2])
    turned = {n: far(t) if n in ("q", "k", "v", "log_decay") else t for n, t in case.items()}
    assert all(turned[n].is_contiguous() and turned[n].stride(1) == 1 << 25 for n in ("q", "k", "v"))
    out, final, tape = ops.linear_attention(**turned, tape=True)
    assert torch.equal(out, want[0]) and torch.equal(final, want[1])
    got = ops.linear_attention_backward(far(go), gs, tape)
    assert all(torch.equal(got[n], grads[n]) for n in grads)
    out, final = ops.linear_attention(**turned)
    assert torch.equal(out, ops.linear_attention(**case)[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_states_off_16_bytes(dtype):
    """A contiguous state that starts anywhere a float may: the same bits as in a state of its own."""
    print(f"case: linear attention state alignment {dtype}", flush=True)
    for width in (64, 20):
        case = make(3, 4, 2, 4, 24, width, dtype)
        token = {n: t[:, 0].contiguous() if n != "state" else t for n, t in case.items()}
        own = case["state"].clone()
        want = ops.linear_attention_step(**dict(token, state=own))
        for start in (1, 2, 3):
            memory = torch.full((case["state"].numel() + 8,), 7.0, device="cuda")
            state = memory[start:start + case["state"].numel()].view(case["state"].shape)
            state.copy_(case["state"])
            out = ops.linear_attention_step(**dict(token, state=state))
            assert torch.equal(out, want) and torch.equal(state, own)
            assert (memory[:start] == 7.0).all() and (memory[start + state.numel():] == 7.0).all()
            state.copy_(case["state"])
            for tape in (False, True):
                got, expected = (ops.linear_attention(**dict(case, state=s), tape=tape) for s in (state, case["state"]))
                assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [5, 100, 700])
@pytest.mark.parametrize("reset", [-float("inf"), -300.0])
def test_an_emptied_state_stays_empty_while_it_grows(reset, T, dtype):
    """Log decays that grow behind one of -inf, or one whose exponential is zero in float32: nothing from before it returns.  No
    later token writes, so answers and state are zeros (e^-220 of what was, which float32 does not hold)."""
    print(f"case: linear attention growth behind {reset}, {T} tokens {dtype}", flush=True)
    case, at = make(2, T, 1, 2, 20, 24, dtype), T // 2
    case["log_decay"][:, at] = reset
    case["log_decay"][:, at + 1:at + 3] = 40.0
    case["k"][:, at:] = 0.0
    for tape in (False, True):
        out, final, *_ = ops.linear_attention(**case, tape=tape)
        assert (out[:, at:] == 0).all() and (final == 0).all()
        assert (out[:, :at] != 0).any()
    check(case, train=False)
