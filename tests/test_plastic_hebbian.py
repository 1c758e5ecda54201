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
