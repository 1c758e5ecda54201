"""Layers with plastic synapses, trained over sequences and run tick by tick: the operators of ``ops`` together.

Spikes pass a dense matrix and a layer norm; from these currents come the queries, keys and values of a gated
delta rule, whose state is the layer's synapses while a sequence runs, and its gates; a dense readout follows.
Training is ``layer_norm`` and ``delta_rule`` with their backward passes, and one ``muon_update`` per dense
matrix; ``PlasticLayer.tick`` continues streams with ``delta_rule_step``.  The dense products are torch's.

``HebbianStack`` has several layers whose synapses only grow and decay, and symbols for inputs: ``embedding`` starts a stream, to
which each layer adds what its ``linear_attention`` answers to the stream's ``rms_norm``, with ``dropout`` while it trains.

``python -m atlas_hip.plastic`` trains one of them (``--rule delta`` or ``hebbian``) to recall: pairs of symbols are shown, then
one symbol of each in another order, and the other is asked for.  It prints one JSON line: the losses, and how far the
ticks' answers are from the sequence's.
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
        out, _, tape = ops.delta_rule(q, k, v, log_decay, beta, scale=1.0, tape=True)
        tensors, ctx.rest = tape.split()
        ctx.save_for_backward(*tensors)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        grads = ops.delta_rule_backward(grad, None, ops.DeltaTape.join(ctx.saved_tensors, ctx.rest))
        return tuple(grads[name] for name in ("q", "k", "v", "log_decay", "beta"))


class RmsNorm(torch.autograd.Function):
    """``ops.rms_norm`` of x added to a stream, for torch's autograd: the normalised stream and the stream."""

    @staticmethod
    def forward(ctx, x, residual, weight):
        y, total, rstd = ops.rms_norm(x, weight, residual, statistics=True)
        ctx.save_for_backward(total, weight, rstd)
        return y, total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_total):
        dx, dweight = ops.rms_norm_backward(grad, *ctx.saved_tensors, grad_total=grad_total)
        return dx, dx, dweight


class LinearAttention(torch.autograd.Function):
    """``ops.linear_attention`` from an empty state, read by queries of length one, for torch's autograd."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay):
        out, _, tape = ops.linear_attention(q, k, v, log_decay, scale=1.0, tape=True)
        tensors, ctx.rest = tape.split()
        ctx.save_for_backward(*tensors)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        grads = ops.linear_attention_backward(grad, None, ops.LinearTape.join(ctx.saved_tensors, ctx.rest))
        return tuple(grads[name] for name in ("q", "k", "v", "log_decay"))


class Embedding(torch.autograd.Function):
    """``ops.embedding`` for torch's autograd."""

    @staticmethod
    def forward(ctx, table, tokens):
        ctx.save_for_backward(tokens)
        ctx.rows = len(table)
        return ops.embedding(table, tokens)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return ops.embedding_backward(grad, *ctx.saved_tensors, ctx.rows), None


class Dropout(torch.autograd.Function):
    """``ops.dropout`` for torch's autograd; a tick on the GPU must not change before the backward pass, which refuses it then."""

    @staticmethod
    def forward(ctx, x, probability, seed, stream, tick):
        held = isinstance(tick, torch.Tensor)
        ctx.arguments = probability, seed, stream, None if held else tick
        ctx.save_for_backward(tick if held else None)
        return ops.dropout(x, probability, seed, stream=stream, tick=tick)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        probability, seed, stream, tick = ctx.arguments
        held, = ctx.saved_tensors
        return ops.dropout(grad, probability, seed, stream=stream, tick=tick if held is None else held), None, None, None, None


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


class HebbianStack:
    """Layers of linear attention on one stream.  Dense matrices are (source, target), float32, in ``matrices``, the
    symbols' rows in ``table``, the norms' weights and the heads' decays (by their logistic function) in ``vectors``."""

    def __init__(self, symbols: int, features: int, heads: int, width: int, outputs: int, *, layers: int = 2,
                 dropout: float = 0.0, seed: int = 0, device="cuda"):
        make = torch.Generator().manual_seed(seed)

        def dense(source, target, size=1.0):
            w = size * torch.randn(source, target, generator=make) / source ** 0.5
            return w.to(device).requires_grad_()

        self.heads, self.width, self.layers, self.dropout, self.seed = heads, width, layers, dropout, seed
        self.table = dense(symbols, features, symbols ** 0.5)
        self.matrices = {f"{name}{layer}": dense(features, heads * width) for layer in range(layers) for name in ("query", "key", "value")}
        self.matrices.update({f"mix{layer}": dense(heads * width, features) for layer in range(layers)})
        self.matrices["readout"] = dense(features, outputs)
        self.vectors = {f"weight{layer}": torch.ones(features, device=device).requires_grad_() for layer in range(layers + 1)}
        self.vectors.update({f"decay{layer}": torch.linspace(2.0, 6.0, heads, device=device).requires_grad_() for layer in range(layers)})
        self.momentum = {name: torch.zeros_like(w, requires_grad=False) for name, w in self.matrices.items()}

    def parts(self, currents, layer: int):
        """q, k, v and the heads' log decays of a layer from its normalised stream (..., features)."""
        shape = (*currents.shape[:-1], self.heads, self.width)
        q, k, v = ((currents @ self.matrices[f"{name}{layer}"]).view(shape) for name in ("query", "key", "value"))
        return F.normalize(q, dim=-1), F.normalize(k, dim=-1), v, F.logsigmoid(self.vectors[f"decay{layer}"])

    def forward(self, tokens, tick=None):
        """Answers (batch, time, outputs) to whole sequences of symbols (batch, time, at once), from empty synapses; a symbol
        that is no row of the table adds nothing.  With a tick (a training step's number) values drop out."""
        stream = Embedding.apply(self.table, tokens).sum(-2)
        added = torch.zeros_like(stream)
        for layer in range(self.layers):
            currents, stream = RmsNorm.apply(added, stream, self.vectors[f"weight{layer}"])
            added = LinearAttention.apply(*self.parts(currents, layer)).flatten(-2) @ self.matrices[f"mix{layer}"]
            if tick is not None and self.dropout:
                added = Dropout.apply(added, self.dropout, self.seed, layer, tick)
        currents, _ = RmsNorm.apply(added, stream, self.vectors[f"weight{self.layers}"])
        return currents @ self.matrices["readout"]

    @torch.no_grad()
    def tick(self, tokens, states):
        """Answers (batch, outputs) to one tick's symbols (batch, at once) of running streams, whose states change in place."""
        stream = ops.embedding(self.table, tokens).sum(-2)
        added = torch.zeros_like(stream)
        for layer, state in enumerate(states):
            currents, stream = ops.rms_norm(added, self.vectors[f"weight{layer}"], stream)
            added = ops.linear_attention_step(*self.parts(currents, layer), state, scale=1.0).flatten(-2) @ self.matrices[f"mix{layer}"]
        return ops.rms_norm(added, self.vectors[f"weight{self.layers}"], stream)[0] @ self.matrices["readout"]

    def states(self, batch: int):
        """Empty synapses of new streams, by layer."""
        shape = (batch, self.heads, self.width, self.width)
        return [torch.zeros(shape, device=self.table.device) for _ in range(self.layers)]

    def train(self, tokens, target, tick, *, learning_rate: float = 0.05):
        """One step on the answers to the last ticks, those of target (batch, ticks); returns the loss before it, on the GPU."""
        parameters = {"table": self.table, **self.matrices, **self.vectors}
        loss = F.cross_entropy(self.forward(tokens, tick)[:, -target.shape[1]:].flatten(0, 1), target.flatten())
        grads = dict(zip(parameters, torch.autograd.grad(loss, list(parameters.values()))))
        with torch.no_grad():
            for name, w in self.matrices.items():
                ops.muon_update(w, grads[name], self.momentum[name], learning_rate=learning_rate)
            for name in ("table", *self.vectors):
                parameters[name].sub_(grads[name], alpha=learning_rate)
        return loss.detach()


def _recall(batch: int, pairs: int, symbols: int, make: torch.Generator):
    """Shown symbols and their partners (batch, pairs), and the order in which they are asked for."""
    shown = torch.rand(batch, symbols, generator=make).argsort(1)[:, :pairs]
    partner = torch.randint(symbols, (batch, pairs), generator=make)
    return shown, partner, torch.rand(batch, pairs, generator=make).argsort(1)


def recall_tokens(batch: int, pairs: int, symbols: int, make: torch.Generator, device="cuda"):
    """As ``recall_batch``, with the symbols in place of their spikes: tokens (batch, 2 pairs, 2) of a table of 2 symbols
    rows, -1 where a half is silent, and the asked symbols (batch, pairs)."""
    shown, partner, order = _recall(batch, pairs, symbols, make)
    tokens = torch.full((batch, 2 * pairs, 2), -1)
    tokens[:, :pairs, 0], tokens[:, :pairs, 1] = shown, partner + symbols
    tokens[:, pairs:, 0] = shown.gather(1, order)
    return tokens.to(device), partner.gather(1, order).to(device)


def recall_batch(batch: int, pairs: int, symbols: int, make: torch.Generator, device="cuda"):
    """Spikes (batch, 2 pairs, 2 symbols) and the asked symbols (batch, pairs).  Of two one-hot halves the first
    ticks show a symbol and its partner; the others show those symbols in another order and ask for the partners."""
    shown, partner, order = _recall(batch, pairs, symbols, make)
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


def run_hebbian(steps: int = 100, batch: int = 256, pairs: int = 24, symbols: int = 32, features: int = 128, heads: int = 2,
                width: int = 64, layers: int = 2, dropout: float = 0.1, seed: int = 0) -> dict:
    make = torch.Generator().manual_seed(seed)
    stack = HebbianStack(2 * symbols, features, heads, width, symbols, layers=layers, dropout=dropout, seed=seed)
    losses = torch.stack([stack.train(*recall_tokens(batch, pairs, symbols, make), step) for step in range(steps)]).tolist()
    tokens, target = recall_tokens(batch, pairs, symbols, make)
    with torch.no_grad():
        whole = stack.forward(tokens)
    states = stack.states(batch)
    ticks = torch.stack([stack.tick(tokens[:, t], states) for t in range(tokens.shape[1])], 1)
    return {"steps": steps, "first_loss": losses[0], "last_loss": losses[-1],
            "recalled": (whole[:, pairs:].argmax(-1) == target).float().mean().item(),
            "ticks_from_sequence": ((ticks - whole).norm() / whole.norm()).item()}


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(prog="python -m atlas_hip.plastic", description="Train plastic layers to recall.")
    for name, value in (("steps", 100), ("batch", 256), ("pairs", 24), ("symbols", 32), ("seed", 0)):
        parser.add_argument(f"--{name}", type=int, default=value)
    parser.add_argument("--rule", choices=("delta", "hebbian"), default="delta", help="one layer of the delta rule, or a Hebbian stack")
    parser.add_argument("--layers", type=int, default=2, help="of the Hebbian stack")
    parser.add_argument("--dropout", type=float, default=0.1, help="of the Hebbian stack while it trains")
    given = parser.parse_args(argv)
    if not 1 <= given.pairs <= given.symbols or given.steps < 1 or given.batch < 1:
        parser.error("steps and batch must be positive, pairs 1 to symbols")
    if given.layers < 1 or not 0.0 <= given.dropout < 1.0:
        parser.error("layers must be positive, dropout 0 or more and below 1")
    if not torch.cuda.is_available():
        print("error: no GPU", file=sys.stderr)
        return 1
    try:
        if given.rule == "hebbian":
            result = run_hebbian(given.steps, given.batch, given.pairs, given.symbols, layers=given.layers, dropout=given.dropout,
                                 seed=given.seed)
        else:
            result = run(given.steps, given.batch, given.pairs, given.symbols, seed=given.seed)
        print(json.dumps(result))
    except (NativeError, NativeUnavailable) as error:
        print(f"error: {error}", file=sys.stderr)
        return 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
