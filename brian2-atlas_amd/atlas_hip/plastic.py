"""A layer with plastic synapses, trained over sequences and run tick by tick: the operators of ``ops`` together.

Spikes pass a dense matrix and a layer norm; from these currents come the queries, keys and values of a gated
delta rule, whose state is the layer's synapses while a sequence runs, and its gates; a dense readout follows.
Training is ``layer_norm`` and ``delta_rule`` with their backward passes, and one ``muon_update`` per dense
matrix; ``PlasticLayer.tick`` continues streams with ``delta_rule_step``.  The dense products are torch's.

``python -m atlas_hip.plastic`` trains it to recall: pairs of symbols are shown, then one symbol of each in
another order, and the other is asked for.  It prints one JSON line: the losses, and how far the ticks' answers are from
the sequence's.
"""
from __future__ import annotations

import argparse
import json
import sys

import torch
import torch.nn.functional as F

from . import ops
from .native import NativeError, NativeUnavailable


class LayerNorm(torch.autograd.Function):
    """``ops.layer_norm`` for torch's autograd."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        y, mean, rstd = ops.layer_norm(x, weight, bias, statistics=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return ops.layer_norm_backward(grad, *ctx.saved_tensors)


class DeltaRule(torch.autograd.Function):
    """``ops.delta_rule`` from an empty state, read by queries of length one, for torch's autograd."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta):
        out, _, ctx.tape = ops.delta_rule(q, k, v, log_decay, beta, scale=1.0, tape=True)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        grads = ops.delta_rule_backward(grad, None, ctx.tape)
        return tuple(grads[name] for name in ("q", "k", "v", "log_decay", "beta"))


class PlasticLayer:
    """Dense matrices are (source, target), float32, in ``matrices``; the norm's weight and bias in ``vectors``."""

    def __init__(self, inputs: int, features: int, heads: int, key: int, value: int, outputs: int, *, seed: int = 0,
                 device="cuda"):
        make = torch.Generator().manual_seed(seed)

        def dense(source, target):
            w = torch.randn(source, target, generator=make) / source ** 0.5
            return w.to(device).requires_grad_()

        self.heads, self.key, self.value = heads, key, value
        self.matrices = {"input": dense(inputs, features), "query": dense(features, heads * key),
                         "key": dense(features, heads * key), "value": dense(features, heads * value),
                         "gates": dense(features, 2 * heads), "readout": dense(heads * value, outputs)}
        self.vectors = {"weight": torch.ones(features, device=device).requires_grad_(),
                        "bias": torch.zeros(features, device=device).requires_grad_()}
        self.momentum = {name: torch.zeros_like(w, requires_grad=False) for name, w in self.matrices.items()}

    def parts(self, currents):
        """q, k, v and the gates from normalised currents (..., features)."""
        w, lead = self.matrices, currents.shape[:-1]
        q = F.normalize((currents @ w["query"]).view(*lead, self.heads, self.key), dim=-1)
        k = F.normalize((currents @ w["key"]).view(*lead, self.heads, self.key), dim=-1)
        v = (currents @ w["value"]).view(*lead, self.heads, self.value)
        gates = (currents @ w["gates"]).view(*lead, 2, self.heads)
        return q, k, v, F.logsigmoid(gates[..., 0, :] + 4.0), torch.sigmoid(gates[..., 1, :])

    def forward(self, spikes):
        """Answers (batch, time, outputs) to whole sequences (batch, time, inputs), from empty synapses."""
        currents = LayerNorm.apply(spikes @ self.matrices["input"], self.vectors["weight"], self.vectors["bias"])
        return DeltaRule.apply(*self.parts(currents)).flatten(-2) @ self.matrices["readout"]

    @torch.no_grad()
    def tick(self, spikes, state):
        """Answers (batch, outputs) to one tick (batch, inputs) of running streams, whose state changes in place."""
        currents = ops.layer_norm(spikes @ self.matrices["input"], self.vectors["weight"], self.vectors["bias"])
        return ops.delta_rule_step(*self.parts(currents), state, scale=1.0).flatten(-2) @ self.matrices["readout"]

    def state(self, batch: int):
        """Empty synapses of new streams."""
        shape = (batch, self.heads, self.key, self.value)
        return torch.zeros(shape, device=self.matrices["input"].device)

    def train(self, spikes, target, *, learning_rate: float = 0.05):
        """One step on the answers to the last ticks, those of target (batch, ticks); returns the loss before it,
        on the GPU."""
        parameters = {**self.matrices, **self.vectors}
        loss = F.cross_entropy(self.forward(spikes)[:, -target.shape[1]:].flatten(0, 1), target.flatten())
        grads = dict(zip(parameters, torch.autograd.grad(loss, list(parameters.values()))))
        with torch.no_grad():
            for name, w in self.matrices.items():
                ops.muon_update(w, grads[name], self.momentum[name], learning_rate=learning_rate)
            for name, w in self.vectors.items():
                w -= learning_rate * grads[name]
        return loss.detach()


def recall_batch(batch: int, pairs: int, symbols: int, make: torch.Generator, device="cuda"):
    """Spikes (batch, 2 pairs, 2 symbols) and the asked symbols (batch, pairs).  Of two one-hot halves the first
    ticks show a symbol and its partner; the others show those symbols in another order and ask for the partners."""
    shown = torch.rand(batch, symbols, generator=make).argsort(1)[:, :pairs]
    partner = torch.randint(symbols, (batch, pairs), generator=make)
    order = torch.rand(batch, pairs, generator=make).argsort(1)
    spikes = torch.zeros(batch, 2 * pairs, 2 * symbols)
    spikes[:, :pairs, :symbols] = F.one_hot(shown, symbols).float()
    spikes[:, :pairs, symbols:] = F.one_hot(partner, symbols).float()
    spikes[:, pairs:, :symbols] = F.one_hot(shown.gather(1, order), symbols).float()
    return spikes.to(device), partner.gather(1, order).to(device)


def run(steps: int = 100, batch: int = 256, pairs: int = 24, symbols: int = 32, features: int = 128, heads: int = 2,
        width: int = 64, seed: int = 0) -> dict:
    make = torch.Generator().manual_seed(seed)
    layer = PlasticLayer(2 * symbols, features, heads, width, width, symbols, seed=seed)
    losses = torch.stack([layer.train(*recall_batch(batch, pairs, symbols, make)) for _ in range(steps)]).tolist()
    spikes, target = recall_batch(batch, pairs, symbols, make)
    with torch.no_grad():
        whole = layer.forward(spikes)
    state = layer.state(batch)
    ticks = torch.stack([layer.tick(spikes[:, t], state) for t in range(spikes.shape[1])], 1)
    return {"steps": steps, "first_loss": losses[0], "last_loss": losses[-1],
            "recalled": (whole[:, pairs:].argmax(-1) == target).float().mean().item(),
            "ticks_from_sequence": ((ticks - whole).norm() / whole.norm()).item()}


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(prog="python -m atlas_hip.plastic", description="Train a plastic layer to recall.")
    for name, value in (("steps", 100), ("batch", 256), ("pairs", 24), ("symbols", 32), ("seed", 0)):
        parser.add_argument(f"--{name}", type=int, default=value)
    given = parser.parse_args(argv)
    if not 1 <= given.pairs <= given.symbols or given.steps < 1 or given.batch < 1:
        parser.error("steps and batch must be positive, pairs 1 to symbols")
    if not torch.cuda.is_available():
        print("error: no GPU", file=sys.stderr)
        return 1
    try:
        print(json.dumps(run(given.steps, given.batch, given.pairs, given.symbols, seed=given.seed)))
    except (NativeError, NativeUnavailable) as error:
        print(f"error: {error}", file=sys.stderr)
        return 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
