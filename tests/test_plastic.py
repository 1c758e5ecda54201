"""The plastic layer: its gradients against the same layer in 64 bits, its ticks against its sequences, and its training."""
import pytest
import torch
import torch.nn.functional as F

from atlas_hip import plastic


def plain(layer, spikes):
    """PlasticLayer.forward token by token in float64 on the CPU; its parameters and the answers."""
    w = {n: t.detach().cpu().double().requires_grad_() for n, t in {**layer.matrices, **layer.vectors}.items()}
    x = spikes.cpu().double() @ w["input"]
    currents = F.layer_norm(x, x.shape[-1:], w["weight"], w["bias"])
    lead = currents.shape[:-1]
    q = F.normalize((currents @ w["query"]).view(*lead, layer.heads, layer.key), dim=-1)
    k = F.normalize((currents @ w["key"]).view(*lead, layer.heads, layer.key), dim=-1)
    v = (currents @ w["value"]).view(*lead, layer.heads, layer.value)
    gates = (currents @ w["gates"]).view(*lead, 2, layer.heads)
    decay, rate = torch.sigmoid(gates[..., 0, :] + 4.0), torch.sigmoid(gates[..., 1, :])
    s = torch.zeros(lead[0], layer.heads, layer.key, layer.value, dtype=torch.float64)
    out = []
    for t in range(lead[1]):
        s = s * decay[:, t, :, None, None]
        e = v[:, t] - (s * k[:, t, ..., None]).sum(-2)
        s = s + rate[:, t, :, None, None] * k[:, t, ..., None] * e[..., None, :]
        out.append((s * q[:, t, ..., None]).sum(-2))
    return w, torch.stack(out, 1).flatten(-2) @ w["readout"]


def test_recall_batch_shows_what_it_asks():
    spikes, target = plastic.recall_batch(7, 5, 9, torch.Generator().manual_seed(1), "cpu")
    assert spikes.shape == (7, 10, 18) and target.shape == (7, 5)
    assert spikes[:, 5:, 9:].sum() == 0
    for sequence, answers in zip(spikes, target):
        for asked, answer in zip(sequence[5:, :9], answers):
            tick = [t for t in range(5) if torch.equal(sequence[t, :9], asked)]
            assert len(tick) == 1 and sequence[tick[0], 9:].argmax() == answer


@pytest.mark.parametrize("given", [["--pairs", "0"], ["--pairs", "33"], ["--steps", "0"], ["--batch", "0"]])
def test_the_command_refuses_sizes(given):
    with pytest.raises(SystemExit):
        plastic.main(given)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs,heads,width", [(5, 2, 16), (35, 1, 24), (65, 3, 40)])
def test_gradients(pairs, heads, width):
    # Every product rounds at 2^-24 of its terms; norms, gates and up to 130 steps of a contracting
    # recurrence let some hundreds of them add up: 1e-4 of each gradient's norm.
    symbols = max(8, pairs)
    spikes, target = plastic.recall_batch(3, pairs, symbols, torch.Generator().manual_seed(2))
    layer = plastic.PlasticLayer(2 * symbols, 48, heads, width, width, symbols)
    w, expected = plain(layer, spikes)
    answers = layer.forward(spikes)
    assert (answers.detach().cpu().double() - expected.detach()).norm() <= 1e-4 * expected.detach().norm()
    own = {**layer.matrices, **layer.vectors}
    grads = torch.autograd.grad(F.cross_entropy(answers[:, pairs:].flatten(0, 1), target.flatten()), list(own.values()))
    wanted = torch.autograd.grad(F.cross_entropy(expected[:, pairs:].flatten(0, 1), target.cpu().flatten()), [w[n] for n in own])
    for name, a, b in zip(own, grads, wanted):
        assert (a.cpu().double() - b).norm() <= 1e-4 * b.norm(), name


@pytest.mark.gpu
def test_ticks_continue_a_sequence_and_training_learns():
    result = plastic.run(steps=60, batch=64, pairs=20, symbols=24)
    assert result["ticks_from_sequence"] <= 1e-4
    assert result["last_loss"] < 0.7 * result["first_loss"]
