"""What the stream, symbol and linear attention operators refuse alike, and their calls from other streams."""
import pytest
import torch
from torch.autograd import forward_ad

from atlas_hip import ops

pytestmark = pytest.mark.gpu


def calls(change):
    """Each operator with one tensor replaced by change(tensor)."""
    g = torch.Generator().manual_seed(0)
    x, m = (torch.randn(4, 32, generator=g).cuda() for _ in range(2))
    k, gate = torch.randn(2, 5, 1, 8, generator=g).cuda(), -torch.rand(2, 5, 1, generator=g).cuda()
    tokens, state = torch.arange(4, device="cuda"), torch.zeros(2, 1, 8, 8, device="cuda")
    rstd = ops.rms_norm(x, statistics=True)[1]
    out, _, tape = ops.linear_attention(k, k, k, gate, tape=True)
    return {"rms_norm": lambda: ops.rms_norm(change(x)), "rms_norm residual": lambda: ops.rms_norm(x, None, change(m)),
            "rms_norm weight": lambda: ops.rms_norm(x, change(x[0].clone())), "rms_norm_8bit": lambda: ops.rms_norm_8bit(change(x)),
            "rms_norm_backward": lambda: ops.rms_norm_backward(change(m), x, None, rstd),
            "rms_norm_backward total": lambda: ops.rms_norm_backward(m, x, None, rstd, grad_total=change(x)),
            "embedding": lambda: ops.embedding(change(x), tokens), "embedding_backward": lambda: ops.embedding_backward(change(x), tokens, 9),
            "dropout": lambda: ops.dropout(change(x), 0.5, 0), "dropout residual": lambda: ops.dropout(x, 0.5, 0, residual=change(m)),
            "linear_attention": lambda: ops.linear_attention(k, k, change(k), gate),
            "linear_attention decay": lambda: ops.linear_attention(k, k, k, change(gate)),
            "linear_attention_step": lambda: ops.linear_attention_step(k[:, 0], k[:, 0], change(k[:, 0]), gate[:, 0], state),
            "linear_attention_backward": lambda: ops.linear_attention_backward(change(out), None, tape)}


def test_tangents_are_refused():
    print("case: dual tensors", flush=True)
    with forward_ad.dual_level():
        for name, call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))).items():
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls(lambda t: t).values():
            call()


def test_negated_views_are_refused():
    print("case: negated views", flush=True)
    for name, call in calls(lambda t: torch.complex(t, -t).conj().imag).items():
        with pytest.raises(ValueError, match="resolve_neg"):
            call()


def test_followed_tensors_are_refused():
    print("case: leaves", flush=True)
    for name, call in calls(lambda t: t.clone().requires_grad_()).items():
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    with torch.no_grad():
        for call in calls(lambda t: t.clone().requires_grad_()).values():
            call()


def everything(case):
    q, gate, grad, tokens, weight = case
    out, final, tape = ops.linear_attention(q, q, q, gate, tape=True)
    grads = ops.linear_attention_backward(grad, final, tape)
    y, total, rstd = ops.rms_norm(out, weight, q, statistics=True)
    dx, dweight = ops.rms_norm_backward(grad, total, weight, rstd, grad_total=q)
    table = ops.embedding_backward(dx.flatten(2), tokens, 40)
    back = ops.embedding(table, tokens)
    return [out, final, *(g for g in grads.values() if g is not None), y, dx, dweight, table, ops.dropout(back, 0.3, 1, residual=back)]


def make(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 500, 2, 48, generator=g).cuda(), -torch.rand(2, 500, 2, generator=g).cuda(), torch.randn(2, 500, 2, 48, generator=g).cuda(),
            torch.randint(-1, 40, (2, 500), generator=g).cuda(), torch.rand(48, generator=g).cuda()]


def test_streams_beside_each_other():
    """Two streams run everything at once, many times, each on its own inputs."""
    print("case: two streams", flush=True)
    cases = [make(1), make(2)]
    want = [everything(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for case, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(everything(case))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_tape_used_on_another_stream():
    print("case: tape on another stream", flush=True)
    q, gate, grad, _, _ = make(3)
    out, final, tape = ops.linear_attention(q, q, q, gate, tape=True)
    want = ops.linear_attention_backward(grad, final, tape)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.linear_attention_backward(grad, final, tape)
    del tape, out
    for _ in range(4):   # memory that the tape gave back must not be taken before the other stream is done
        torch.full((2, 500, 2, 48, 48), 7.0, device="cuda")
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(got[n], want[n]) for n in want if want[n] is not None)


def test_inputs_stay_as_they_are():
    print("case: inputs", flush=True)
    case = make(4)
    copies = [t.clone() for t in case]
    everything(case)
    assert all(torch.equal(a, b) for a, b in zip(case, copies))
    x = case[0]
    same = ops.rms_norm(x, None, x)   # a tensor that is its own residual
    assert torch.equal(same[1], x + x)
    assert torch.equal(ops.dropout(x, 0.5, 0, residual=x), ops.dropout(x, 0.5, 0) + x)
