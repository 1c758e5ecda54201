"""The Hebbian stack: its gradients against the same stack in 64 bits, dropout among them, its ticks against its sequences,
and the operators together in a captured step."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from atlas_hip import ops, plastic
from oracle import ops_oracle as oo


def plain(stack, tokens, tick=None):
    """HebbianStack.forward token by token in float64 on the CPU; its parameters and the answers."""
    given = {"table": stack.table, **stack.matrices, **stack.vectors}
    w = {n: t.detach().cpu().double().requires_grad_() for n, t in given.items()}
    tokens = tokens.cpu()
    known = (tokens >= 0) & (tokens < len(w["table"]))
    stream = (w["table"][tokens.clamp(0, len(w["table"]) - 1)] * known[..., None]).sum(-2)

    def norm(x, weight):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight

    lead = stream.shape[:-1]
    for layer in range(stack.layers):
        currents = norm(stream, w[f"weight{layer}"])
        q, k, v = ((currents @ w[f"{n}{layer}"]).view(*lead, stack.heads, stack.width) for n in ("query", "key", "value"))
        q, k, decay = F.normalize(q, dim=-1), F.normalize(k, dim=-1), torch.sigmoid(w[f"decay{layer}"])
        s = torch.zeros(lead[0], stack.heads, stack.width, stack.width, dtype=torch.float64)
        out = []
        for t in range(lead[1]):
            s = decay[:, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
            out.append((s * q[:, t, :, :, None]).sum(-2))
        added = torch.stack(out, 1).flatten(-2) @ w[f"mix{layer}"]
        if tick is not None:
            kept = oo.dropout_kept(added.numel(), stack.dropout, stack.seed, layer, tick)
            added = added * torch.from_numpy(kept).view(added.shape) / (1.0 - stack.dropout)
        stream = stream + added
    return w, norm(stream, w[f"weight{stack.layers}"]) @ w["readout"]


def test_tokens_are_the_batchs_spikes():
    spikes, target = plastic.recall_batch(7, 5, 9, torch.Generator().manual_seed(1), "cpu")
    tokens, asked = plastic.recall_tokens(7, 5, 9, torch.Generator().manual_seed(1), "cpu")
    assert torch.equal(target, asked)
    shown = F.one_hot(tokens.clamp(min=0), 18) * (tokens >= 0)[..., None]
    assert torch.equal(shown.sum(2).float(), spikes)


@pytest.mark.parametrize("given", [["--rule", "hebbian", "--layers", "0"], ["--rule", "hebbian", "--dropout", "1"], ["--dropout", "-0.1"], ["--rule", "other"]])
def test_the_command_refuses(given):
    with pytest.raises(SystemExit):
        plastic.main(given)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs,heads,width,tick", [(5, 2, 16, None), (35, 1, 24, 7), (65, 3, 40, 1)])
def test_gradients(pairs, heads, width, tick):
    # Every product rounds at 2^-24 of its terms; two layers of norms and up to 130 ticks of sums let some hundreds of them
    # add up: 1e-4 of each gradient's norm.
    symbols = max(8, pairs)
    tokens, target = plastic.recall_tokens(3, pairs, symbols, torch.Generator().manual_seed(2))
    stack = plastic.HebbianStack(2 * symbols, 48, heads, width, symbols, dropout=0.3, seed=5)
    w, expected = plain(stack, tokens, tick)
    answers = stack.forward(tokens, tick)
    assert (answers.detach().cpu().double() - expected.detach()).norm() <= 1e-4 * expected.detach().norm()
    own = {"table": stack.table, **stack.matrices, **stack.vectors}
    grads = torch.autograd.grad(F.cross_entropy(answers[:, pairs:].flatten(0, 1), target.flatten()), list(own.values()))
    wanted = torch.autograd.grad(F.cross_entropy(expected[:, pairs:].flatten(0, 1), target.cpu().flatten()), [w[n] for n in own])
    for name, a, b in zip(own, grads, wanted):
        assert (a.cpu().double() - b).norm() <= 1e-4 * b.norm(), name


@pytest.mark.gpu
def test_ticks_continue_a_sequence():
    result = plastic.run_hebbian(steps=3, batch=16, pairs=20, symbols=24)
    assert result["ticks_from_sequence"] <= 1e-4 and np.isfinite([result["first_loss"], result["last_loss"]]).all()


@pytest.mark.gpu
def test_the_operators_in_a_captured_step():
    """A step of all operators, forwards and backwards, recorded once: replays on other inputs and ticks, with eager work and
    waits between them, are the eager calls' results."""
    print("case: captured step", flush=True)
    make = torch.Generator().manual_seed(3)
    normal = lambda *shape: torch.randn(shape, generator=make).cuda()  # noqa: E731
    B, T, H, d, rows = 2, 300, 2, 32, 50
    static = {"tokens": torch.randint(-1, rows, (B, T), generator=make).cuda(), "table": normal(rows, H * d), "weight": normal(H * d),
              "decay": -torch.rand(H, generator=make).cuda(), "grad": normal(B, T, H, d), "tick": torch.zeros(1, dtype=torch.int64, device="cuda"),
              "state": normal(B, H, d, d)}

    def step(s):
        x = ops.embedding(s["table"], s["tokens"], scale=2.0)
        y, total, rstd = ops.rms_norm(ops.dropout(x, 0.2, 9, stream=1, tick=s["tick"]), s["weight"], x, statistics=True)
        values, scale = ops.rms_norm_8bit(total, s["weight"])
        q = y.view(B, T, H, d)
        out, final, tape = ops.linear_attention(q, q, q, s["decay"], s["state"], tape=True)
        grads = ops.linear_attention_backward(s["grad"], final, tape)
        g = (grads["q"] + grads["k"] + grads["v"]).flatten(-2)
        dx, dweight = ops.rms_norm_backward(g, total, s["weight"], rstd, grad_total=g)
        back = ops.dropout(dx, 0.2, 9, stream=1, tick=s["tick"], residual=dx)
        table = ops.embedding_backward(back, s["tokens"], rows, scale=2.0)
        after = ops.linear_attention_step(q[:, 0], q[:, 1], q[:, 2], s["decay"], final)
        return [y, total, values.float(), scale, out, final, after, grads["log_decay"], grads["state"], dweight, table]

    step(static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        results = step(static)
    masks = []
    for replay in range(4):
        static["tick"].fill_(replay)
        static["tokens"].copy_(torch.randint(-1, rows, (B, T), generator=make).cuda())
        static["state"].copy_(normal(B, H, d, d))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        for a, b in zip(got, step(static)):
            assert torch.equal(a, b), replay
        masks.append(got[1])
        torch.cuda.synchronize()
    assert not torch.equal(masks[0], masks[1])


# What each autograd function keeps, with the inputs of a call (the last two: not followed)
def functions():
    g = torch.Generator().manual_seed(6)
    normal = lambda *shape: torch.randn(shape, generator=g).cuda()  # noqa: E731
    q, k, v = (normal(2, 70, 2, 16) for _ in range(3))
    gate = -torch.rand(2, 70, 2, generator=g).cuda()
    beta, decay = torch.rand(2, 70, 2, generator=g).cuda(), -torch.rand(2, generator=g).cuda()
    return {"LinearAttention": (q, k, v, gate), "LinearAttention by head": (q, k, v, decay), "LinearAttention without": (q, k, v, None),
            "DeltaRule": (q, F.normalize(k, dim=-1), v, gate, beta),
            "LayerNorm": (normal(9, 24), normal(24), normal(24)), "RmsNorm": (normal(9, 24), normal(9, 24), normal(24)),
            "Dropout": (normal(9, 24), 0.3, 5, 2, torch.full((1,), 4, device="cuda"))}


def called(name, given):
    leaves = [t.clone().requires_grad_() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for t in given]
    inputs = [t.view_as(t) if isinstance(t, torch.Tensor) else t for t in leaves]   # what may change in place
    out = getattr(plastic, name.split()[0]).apply(*inputs)
    return [t for t in leaves if isinstance(t, torch.Tensor) and t.requires_grad], inputs, out if isinstance(out, torch.Tensor) else out[0]


NAMES = ["LinearAttention", "LinearAttention by head", "LinearAttention without", "DeltaRule", "LayerNorm", "RmsNorm", "Dropout"]
KEPT = {"LinearAttention": range(4), "LinearAttention by head": range(4), "LinearAttention without": range(3), "DeltaRule": range(5),
        "LayerNorm": (0, 1), "RmsNorm": (2,), "Dropout": (4,)}


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_inputs_that_changed_before_the_backward_pass_are_refused(name):
    print(f"case: changed inputs of {name}", flush=True)
    given = functions()[name]
    for at in KEPT[name]:
        leaves, inputs, out = called(name, given)
        with torch.no_grad():
            inputs[at].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaves, allow_unused=True)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_are_autograds(name):
    """Their hooks see them and may lay them out anew, a second backward pass is refused unless they are kept, and their
    memory goes with the graph."""
    print(f"case: saved tensors of {name}", flush=True)
    given = functions()[name]
    leaves, _, out = called(name, given)
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(8)).cuda()
    want = torch.autograd.grad(out, leaves, grad, allow_unused=True, retain_graph=True)
    again = torch.autograd.grad(out, leaves, grad, allow_unused=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(want, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, grad, allow_unused=True)
    seen = []

    def pack(t):
        seen.append(t)
        return t.detach().cpu(), t.stride()

    def unpack(kept):   # in other memory, and of other strides where there is more than one axis
        t = kept[0].cuda()
        return t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() > 2 else t

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        leaves, _, out = called(name, given)
    assert len(seen) >= len(KEPT[name])
    got = torch.autograd.grad(out, leaves, grad, allow_unused=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["LinearAttention", "DeltaRule"])
def test_the_tapes_memory_goes_with_the_graph(name):
    print(f"case: memory of {name}", flush=True)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(2, 3000, 2, 64, generator=g).cuda()
    gate = -torch.rand(2, 3000, 2, generator=g).cuda()
    given = (q, q, q, gate) if name == "LinearAttention" else (q, F.normalize(q, dim=-1), q, gate, gate.exp())
    leaves, inputs, out = called(name, given)
    del inputs
    requested = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731
    before = requested()
    grads = torch.autograd.grad(out.sum(), leaves)
    tape = 2 * 2 * 64 * 64 * 4   # the final states alone
    assert requested() - before <= sum(t.numel() * t.element_size() for t in grads) - tape, "out still lives, its graph's tape does not"


@pytest.mark.gpu
def test_tapes_of_other_tensors_are_refused():
    print("case: tapes of other tensors", flush=True)
    q, gate = torch.randn(2, 300, 2, 16, device="cuda"), -torch.rand(2, 300, 2, device="cuda")
    for rule, cls in ((lambda *a: ops.linear_attention(*a, tape=True)[2], ops.LinearTape), (lambda *a: ops.delta_rule(*a, gate.exp(), tape=True)[2], ops.DeltaTape)):
        tensors, rest = rule(q, q, q, gate).split()
        for at, other in ((0, q[:, :299]), (2, q.bfloat16()), (-1, tensors[-1][:-64]), (-1, tensors[-1].float()), (-1, tensors[-1][::2]), (-1, None)):
            changed = list(tensors)
            changed[at] = other
            with pytest.raises(ValueError):
                cls.join(changed, rest)
        for wrong in (lambda: cls.join(tensors[:-1], rest), lambda: cls.join((), rest)):
            with pytest.raises(ValueError):
                wrong()


@pytest.mark.gpu
def test_tapes_of_tensors_laid_out_anew():
    """With a state, lengths and a scale: the same gradients, bit by bit."""
    print("case: tapes laid out anew", flush=True)
    g = torch.Generator().manual_seed(9)
    q, gate, state = torch.randn(2, 300, 2, 16, generator=g).cuda(), -torch.rand(2, 300, 2, generator=g).cuda(), torch.randn(2, 2, 16, 16, generator=g).cuda()
    lengths = torch.tensor([300, 77], dtype=torch.int32, device="cuda")
    for rule, back, cls in ((ops.linear_attention, ops.linear_attention_backward, ops.LinearTape), (ops.delta_rule, ops.delta_rule_backward, ops.DeltaTape)):
        gates = (gate,) if cls is ops.LinearTape else (gate, gate.exp())
        out, final, tape = rule(F.normalize(q, dim=-1), F.normalize(q.flip(1), dim=-1), q, *gates, state, lengths=lengths, scale=0.3, tape=True)
        want = back(out, final, tape)
        tensors, rest = tape.split()
        turned = [t if t is None or t.dim() < 3 else t.transpose(-1, 1).contiguous().transpose(-1, 1) for t in tensors]
        assert not turned[5].is_contiguous()
        off = torch.cat([tensors[-1][:3], tensors[-1]])[3:]   # memory that starts anywhere
        for memory in (tensors[-1], off):
            got = back(out, final, cls.join([*turned[:-1], memory], rest))
            assert all(a is b is None or torch.equal(a, b) for a, b in zip(want.values(), got.values()))
