"""More operators of ``atlas_hip.ops`` as measurable cases, those of a layer whose inputs are symbols and whose
synapses learn by Hebb's rule: the embedding of symbols with its gradient, root-mean-square normalisation of a residual
stream (also to 8 bits), dropout from the simulator's counter generator, and linear attention with a decay per head.

Sizes come from the recurrent trainer's plan (256 hidden, 100 ticks, batch 256), the recall task (32 symbols, 48 ticks)
or are generic.  ``run`` computes each operator in a plain form of elementary torch operations in float32 (sums of log
decays and what is rounded to 8 bits in float64), rounded once at the end; with ``own`` set it calls the framework.
``exact`` is the same from the operators' definitions in float64: linear attention token by token, its gradients by the
reversed recurrence.
"""
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
LARGEST = 448.0                              # of the 8-bit type, e4m3
SEED, STREAM, RATE = 20240607, 3, 0.1        # of dropout
SCALE = 16.0                                 # of embeddings
CHUNK = 64                                   # tokens per chunk of the plain linear attention


def listed():
    return [
        # one tick's currents of the trainer's batch added to their stream: launch latency counts
        {"name": "rms_tick", "kind": "rms", "rows": 256, "width": 256, "type": "f32", "residual": True},
        # odd rows of an odd width, trained: no vector access is aligned
        {"name": "rms_train_odd", "kind": "rms_train", "rows": 9973, "width": 1023, "type": "bf16", "residual": False},
        # a wide residual stream over a large batch, trained: memory bandwidth
        {"name": "rms_train_wide", "kind": "rms_train", "rows": 16384, "width": 4096, "type": "bf16", "residual": True},
        # the input of an 8-bit product while serving a batch
        {"name": "rms_8bit_batch", "kind": "rms_8bit", "rows": 2048, "width": 4096, "type": "bf16", "residual": True},
        # a whole batch of the trainer's hidden layer, 100 ticks of 256 samples: forward and gradient
        {"name": "dropout_train_ticks", "kind": "dropout_train", "rows": 25600, "width": 256, "type": "f32"},
        # a wide layer of odd rows added to its stream
        {"name": "dropout_odd", "kind": "dropout", "rows": 12289, "width": 4099, "type": "bf16"},
        # the recall task's symbols: few rows, each met hundreds of times
        {"name": "embed_train_symbols", "kind": "embed_train", "rows": 32, "width": 128, "batch": 256, "time": 48, "type": "f32",
         "padded": False},
        # a large table, of which a padded batch meets a part, the frequent symbols often
        {"name": "embed_train_large", "kind": "embed_train", "rows": 50000, "width": 1024, "batch": 16, "time": 2047, "type": "bf16",
         "padded": True},
        # streaming: one tick of 64 streams, a state of 128 x 128 for each of 8 heads
        {"name": "linear_tick", "kind": "linear_step", "batch": 64, "heads": 8, "value_heads": 8, "key": 128, "value": 128,
         "type": "bf16", "decay": "head"},
        # the trainer's batch and ticks through 256 units as 4 heads of 64: forward and backward
        {"name": "linear_train_ticks", "kind": "linear_train", "batch": 256, "time": 100, "heads": 4, "value_heads": 4, "key": 64,
         "value": 64, "type": "f32", "ragged": False, "state": False, "decay": "head"},
        # one long recording through a wide layer: few rows, a long axis
        {"name": "linear_long", "kind": "linear", "batch": 1, "time": 16384, "heads": 16, "value_heads": 16, "key": 128,
         "value": 128, "type": "bf16", "ragged": False, "state": True, "decay": "token"},
        # training over recordings that end at different ticks, keys shared by four value heads
        {"name": "linear_train_shared", "kind": "linear_train", "batch": 2, "time": 4099, "heads": 4, "value_heads": 16, "key": 128,
         "value": 96, "type": "bf16", "ragged": True, "state": True, "decay": "token"},
    ]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    kind = rng.choice(["rms", "rms_train", "rms_8bit", "dropout", "dropout_train", "embed", "embed_train", "linear_step", "linear",
                       "linear_train"])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16"])}
    if kind.startswith("rms") or kind.startswith("dropout"):
        width = spread(20, 8192)
        case.update(rows=spread(1, min(65536, (1 << 25) // width)), width=width)
        if kind.startswith("rms"):
            case["residual"] = rng.random() < 0.5
        return case
    if kind.startswith("embed"):
        width = spread(16, 2048)
        case.update(rows=spread(16, min(100000, (1 << 25) // width)), width=width)
        case["time"] = spread(1, min(4096, (1 << 24) // width))
        case.update(batch=spread(1, min(256, (1 << 24) // (width * case["time"]))), padded=rng.random() < 0.5)
        return case
    heads = spread(1, 8)
    case.update(batch=0, heads=heads, value_heads=heads * rng.choice([1, 1, 2, 4]),
                key=rng.choice([16, 32, 40, 64, 96, 128, spread(8, 128)]),
                value=rng.choice([16, 32, 64, 96, 128, spread(8, 128)]), decay=rng.choice(["token", "head"]))
    if kind == "linear_step":
        case["batch"] = spread(1, max(1, 512 // case["value_heads"]))
        return case
    case["time"] = spread(1, 8192)
    most = max(1, (1 << 16) // (case["time"] * case["value_heads"]))
    case.update(batch=spread(1, min(most, 256)), ragged=rng.random() < 0.5, state=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    device = torch.device("cuda")
    random = torch.Generator(device=device)
    random.manual_seed(seed)
    dtype, kind = TYPES[case["type"]], case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=random, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=random, device=device)

    state = {"case": case}
    if kind.startswith("rms") or kind.startswith("dropout"):
        rows, width = case["rows"], case["width"]
        # currents: units of their own mean and size, a sample's drive common to its units
        x = normal(rows, width) * (0.5 + uniform(width)) + 0.3 * normal(width) + 0.5 * normal(rows, 1)
        state["x"] = x.to(dtype)
        state["residual"] = (2.0 * normal(rows, width)).to(dtype) if case.get("residual", kind == "dropout") else None
        state["grad"] = normal(rows, width).to(dtype)
        if kind.startswith("rms"):
            state["weight"] = 1.0 + 0.1 * normal(width)
            state["grad_total"] = normal(rows, width).to(dtype) if case["residual"] else None
        else:
            # the training step's number, on the GPU, where a captured step counts it up
            state["tick"] = torch.full((1,), seed % 1000003, dtype=torch.int64, device=device)
    elif kind.startswith("embed"):
        rows, lead = case["rows"], (case["batch"], case["time"])
        state["table"] = (normal(rows, case["width"]) / SCALE).to(dtype)
        # the r-th most frequent symbol is met in proportion to 1 / r
        tokens = (torch.exp(uniform(*lead).double() * math.log(rows + 1.0)) - 1.0).long().clamp(0, rows - 1)
        if case["padded"]:
            ends = torch.randint(0, case["time"] + 1, (case["batch"], 1), generator=random, device=device)
            tokens = tokens.masked_fill(torch.arange(case["time"], device=device) >= ends, -1)
        state["tokens"] = tokens
        state["grad"] = (1e-2 * normal(*lead, case["width"])).to(dtype)
    else:
        B, H, Hv, dk, dv = case["batch"], case["heads"], case["value_heads"], case["key"], case["value"]
        lead = (B,) if kind == "linear_step" else (B, case["time"])
        # keys and queries of unit length, half of them along a common direction as firing rates are
        common = normal(dk).abs()
        q, k = (normal(*lead, H, dk) + 0.5 * common for _ in range(2))
        state["q"], state["k"] = ((a / a.norm(dim=-1, keepdim=True)).to(dtype) for a in (q, k))
        state["v"] = normal(*lead, Hv, dv).to(dtype)
        # decays from a few ticks to thousands
        shape = (Hv,) if case["decay"] == "head" else (*lead, Hv)
        state["log_decay"] = -torch.exp(-7.0 + 6.0 * uniform(*shape))
        if kind == "linear_step" or case["state"]:
            state["state"] = 0.3 * normal(B, Hv, dk, dv)
        if kind != "linear_step":
            state["lengths"] = None
            if case["ragged"]:
                state["lengths"] = torch.randint(0, case["time"] + 1, (B,), generator=random, device=device,
                                                 dtype=torch.int32)
                state["lengths"][0] = case["time"]
        if kind == "linear_train":
            state["grad"] = normal(*lead, Hv, dv).to(dtype)
            state["grad_state"] = 0.1 * normal(B, Hv, dk, dv)
    return state


# ------------------------------------------------------------------------------------- plain forms
def _plain_rms(s):
    kind, dtype = s["case"]["kind"], s["x"].dtype
    total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype)
    result = {} if s["residual"] is None else {"total": total}
    if kind == "rms_8bit":
        t = total.double()
        y = t * torch.rsqrt(t.square().mean(dim=-1, keepdim=True) + EPS) * s["weight"].double()
        scale = (y.abs().amax(dim=-1) / LARGEST).clamp(min=2.0 ** -126)
        result.update(values=(y / scale[:, None]).float().to(torch.float8_e4m3fn), scale=scale.float())
        return result
    t = total.float()
    rstd = torch.rsqrt(t.square().mean(dim=-1, keepdim=True) + EPS)
    normed = t * rstd
    result["y"] = (normed * s["weight"]).to(dtype)
    if kind == "rms_train":
        grad = s["grad"].float()
        scaled = grad * s["weight"]
        dx = rstd * (scaled - normed * (scaled * normed).mean(dim=-1, keepdim=True))
        dx = dx if s["grad_total"] is None else dx + s["grad_total"].float()
        result.update(x=dx.to(dtype), weight=(grad * normed).sum(dim=0))
    return result


def _kept(shape, tick):
    """Where dropout keeps its values: element i takes 32 bits of draw i // 2, the low ones where i is even, and is
    dropped where they are below the rate's share of 2^32.  Draw n: splitmix64's finaliser of
    seed ^ stream C1 ^ tick C2 ^ n C3, in 64-bit integers that wrap round."""
    def signed(c):
        return c - (1 << 64) if c >> 63 else c

    def mixed(v, shift, factor):
        return (v ^ ((v >> shift) & ((1 << (64 - shift)) - 1))) * signed(factor)

    count = math.prod(shape)
    index = torch.arange((count + 1) // 2, dtype=torch.int64, device=tick.device)
    v = (SEED ^ signed(STREAM * 0x9E3779B97F4A7C15 % (1 << 64))) ^ (tick * signed(0xD1B54A32D192ED03)) ^ (index * signed(0x94D049BB133111EB))
    v = mixed(mixed(v, 30, 0xBF58476D1CE4E5B9), 27, 0x94D049BB133111EB)
    v = v ^ ((v >> 31) & 0x1FFFFFFFF)
    bits = torch.stack([v & 0xFFFFFFFF, (v >> 32) & 0xFFFFFFFF], dim=1).flatten()[:count]
    return (bits >= round(RATE * 2.0 ** 32)).view(shape)


def _plain_dropout(s):
    factor = _kept(s["x"].shape, s["tick"]) * (1.0 / (1.0 - RATE))
    y = s["x"].float() * factor
    y = y if s["residual"] is None else y + s["residual"].float()
    result = {"y": y.to(s["x"].dtype)}
    if s["case"]["kind"] == "dropout_train":
        result["x"] = (s["grad"].float() * factor).to(s["x"].dtype)
    return result


def _plain_embed(s):
    table, tokens = s["table"], s["tokens"]
    known = (tokens >= 0)[..., None]
    at = tokens.clamp(min=0)
    result = {"out": (table[at].float() * (SCALE * known)).to(table.dtype)}
    if s["case"]["kind"] == "embed_train":
        grad = (s["grad"].float() * (SCALE * known)).flatten(0, 1)
        result["table"] = torch.zeros_like(table, dtype=torch.float32).index_add_(0, at.flatten(), grad).to(table.dtype)
    return result


def _plain_linear_step(s):
    group = s["v"].shape[1] // s["q"].shape[1]
    q, k = (s[n].float().repeat_interleave(group, dim=1) for n in ("q", "k"))
    state = s["state"]
    state.mul_(torch.exp(s["log_decay"])[..., None, None])
    state.add_(k[..., :, None] * s["v"].float()[..., None, :])
    out = torch.matmul(q[..., None, :], state)[..., 0, :] / math.sqrt(q.shape[-1])
    return {"out": out.to(s["v"].dtype), "state": state}


def _chunked_linear(q, k, v, log_decay, state, lengths):
    """Chunks of CHUNK tokens: decayed products of queries and keys within a chunk, and what the chunks before it left,
    whose own sums are joined by one product with the decays between chunks."""
    B, T, Hv, dv = v.shape
    group, dk = Hv // q.shape[2], q.shape[3]
    log_decay = log_decay.double().expand(B, T, Hv)
    live = torch.ones(1, 1, 1, device=v.device)
    if lengths is not None:
        live = (torch.arange(T, device=v.device) < lengths[:, None]).float()[..., None]
        log_decay, k = log_decay * live, k * live[..., None]
    chunks = -(-T // CHUNK)
    pad = chunks * CHUNK - T

    def split(a):  # (batch, time, heads, ...) -> (batch, heads, chunks, CHUNK, ...)
        a = torch.cat([a, a.new_zeros(B, pad, *a.shape[2:])], dim=1) if pad else a
        return a.reshape(B, chunks, CHUNK, *a.shape[2:]).movedim(3, 1).contiguous()

    q, k, v, g = split(q), split(k), split(v), split(log_decay).cumsum(dim=-1)
    q, k = (a.repeat_interleave(group, dim=1) for a in (q, k))
    index = torch.arange(CHUNK, device=v.device)
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(index > index[:, None], -math.inf)).float()
    since, rest = torch.exp(g).float()[..., None], torch.exp(g[..., -1:] - g).float()[..., None]
    ends = torch.cat([g.new_zeros(B, Hv, 1), g[..., -1].cumsum(dim=-1)], dim=-1)      # log decay before each chunk, after all
    order = torch.arange(chunks + 1, device=v.device)
    between = ends[..., :, None] - ends[..., None, 1:]                                # from each chunk's end to each start
    between = torch.exp(between.masked_fill(order[:-1] >= order[:, None], -math.inf)).float()
    own_sums = torch.matmul((rest * k).transpose(-2, -1), v)
    states = torch.matmul(between, own_sums.flatten(-2)).unflatten(-1, (dk, dv))
    if state is not None:
        states = states + torch.exp(ends).float()[..., None, None] * state[:, :, None]
    out = torch.matmul(since * q, states[:, :, :-1]) + torch.matmul(decay * torch.matmul(q, k.transpose(-2, -1)), v)
    out = out.movedim(1, 3).reshape(B, chunks * CHUNK, Hv, dv)[:, :T] * (live[..., None] / math.sqrt(dk))
    return out, states[:, :, -1]


def _plain_linear(s):
    train = "grad" in s
    names = ["q", "k", "v", "log_decay"] + (["state"] if "state" in s else [])
    leaves = {n: s[n].float().detach().requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        out, state = _chunked_linear(*(leaves.get(n) for n in ("q", "k", "v", "log_decay", "state")), s["lengths"])
        rounded = {"out": out.detach().to(s["v"].dtype), "state": state.detach()}
        if train:
            grads = torch.autograd.grad([out, state], list(leaves.values()), [s["grad"].float(), s["grad_state"]])
            rounded.update({"grad_" + n: g.to(s[n].dtype) for n, g in zip(names, grads)})
    return rounded


# ------------------------------------------------------------------------------------------- a pass
def _ops():
    if str(ROOT / "brian2-atlas_amd") not in sys.path:
        sys.path.insert(0, str(ROOT / "brian2-atlas_amd"))
    from atlas_hip import ops
    return ops


def _own(s):
    ops, kind = _ops(), s["case"]["kind"]
    if kind == "rms_8bit":
        names = ("values", "scale") if s["residual"] is None else ("values", "scale", "total")
        return dict(zip(names, ops.rms_norm_8bit(s["x"], s["weight"], s["residual"], eps=EPS)))
    if kind == "rms":
        y = ops.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        return {"y": y} if s["residual"] is None else {"y": y[0], "total": y[1]}
    if kind == "rms_train":
        y, *total, rstd = ops.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS, statistics=True)
        dx, dw = ops.rms_norm_backward(s["grad"], total[0] if total else s["x"], s["weight"], rstd, grad_total=s["grad_total"])
        result = {"y": y, "x": dx, "weight": dw}
        return {**result, "total": total[0]} if total else result
    if kind.startswith("dropout"):
        where = {"stream": STREAM, "tick": s["tick"]}
        result = {"y": ops.dropout(s["x"], RATE, SEED, residual=s["residual"], **where)}
        if kind == "dropout_train":
            result["x"] = ops.dropout(s["grad"], RATE, SEED, **where)
        return result
    if kind.startswith("embed"):
        result = {"out": ops.embedding(s["table"], s["tokens"], scale=SCALE)}
        if kind == "embed_train":
            result["table"] = ops.embedding_backward(s["grad"], s["tokens"], s["case"]["rows"], scale=SCALE)
        return result
    inputs = [s[n] for n in ("q", "k", "v", "log_decay")]
    if kind == "linear_step":
        return {"out": ops.linear_attention_step(*inputs, s["state"]), "state": s["state"]}
    if kind == "linear":
        out, state = ops.linear_attention(*inputs, s.get("state"), lengths=s["lengths"])
        return {"out": out, "state": state}
    out, state, tape = ops.linear_attention(*inputs, s.get("state"), lengths=s["lengths"], tape=True)
    grads = ops.linear_attention_backward(s["grad"], s["grad_state"], tape)
    result = {"out": out, "state": state}
    result.update({"grad_" + n: g for n, g in grads.items() if g is not None})
    return result


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind.startswith("rms"):
        return _plain_rms(state)
    if kind.startswith("dropout"):
        return _plain_dropout(state)
    if kind.startswith("embed"):
        return _plain_embed(state)
    return _plain_linear_step(state) if kind == "linear_step" else _plain_linear(state)


def work(case):
    size, kind = 4 if case["type"] == "f32" else 2, case["kind"]
    if kind.startswith("rms"):
        n, w, rows = case["rows"] * case["width"], case["width"], case["rows"]
        stream = 2 * n * size if case["residual"] else 0                       # the residual and the total
        if kind == "rms_8bit":
            return {"bytes": n * (size + 1) + stream + 4 * w + 4 * rows, "flops": 8 * n}
        if kind == "rms":
            return {"bytes": 2 * n * size + stream + 4 * w, "flops": 5 * n}
        grad_total = n * size if case["residual"] else 0
        return {"bytes": 4 * n * size + stream + grad_total + 8 * w, "flops": 14 * n}
    if kind.startswith("dropout"):
        n = case["rows"] * case["width"]
        return {"bytes": (4 if kind == "dropout_train" else 3) * n * size, "flops": 10 * n}
    if kind.startswith("embed"):
        tokens, w = case["batch"] * case["time"], case["width"]
        met = min(tokens, case["rows"])                                        # rows of the table that can be met
        look = met * w * size + tokens * (w * size + 8)
        if kind == "embed":
            return {"bytes": look, "flops": tokens * w}
        return {"bytes": look + tokens * w * size + case["rows"] * w * size, "flops": 3 * tokens * w}
    tokens, Hv = case["batch"] * case.get("time", 1), case["value_heads"]
    qk, v = tokens * case["heads"] * case["key"], tokens * Hv * case["value"]
    cells, gates = case["batch"] * Hv * case["key"] * case["value"], tokens * Hv if case["decay"] == "token" else Hv
    if kind == "linear_step":
        return {"bytes": size * (2 * qk + 2 * v) + 4 * gates + 8 * cells, "flops": 5 * cells}
    given = 4 * cells * (2 if case["state"] else 1)
    if kind == "linear":
        return {"bytes": size * (2 * qk + 2 * v) + 4 * gates + given, "flops": 4 * tokens * Hv * case["key"] * case["value"]}
    return {"bytes": size * (4 * qk + 4 * v) + 8 * gates + 2 * given,
            "flops": 14 * tokens * Hv * case["key"] * case["value"]}


# -------------------------------------------------------------------------------- exact, in 64 bits
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]

    def rms():
        x = s["x"].double()
        result = {}
        if s["residual"] is not None:
            # the stream is rounded before the norm reads it, and that rounding is part of the definition
            x = x + s["residual"].double()
            result["total"] = x
            x = x.to(s["x"].dtype).double()
        sigma = torch.sqrt((x * x).sum(1, keepdim=True) / case["width"] + EPS)
        z, w = x / sigma, s["weight"].double()
        y = z * w
        if kind == "rms_8bit":
            scale = (y.abs().max(dim=1).values / LARGEST).clamp(min=2.0 ** -126)
            result.update(values=y / scale[:, None], scale=scale)
            return result
        result["y"] = y
        if kind == "rms_train":
            g = s["grad"].double()
            h = g * w
            result["x"] = (h - z * ((h * z).sum(1, keepdim=True) / case["width"])) / sigma
            if s["grad_total"] is not None:
                result["x"] = result["x"] + s["grad_total"].double()
            result["weight"] = (g * z).sum(0)
        return result

    def dropout():
        # the draws as unsigned numbers in two halves of 32 bits each, products by long multiplication
        low = 0xFFFFFFFF

        def times(a, c):
            (ah, al), (ch, cl) = a, (c >> 32, c & low)
            middle = (al * (cl >> 16) & low) << 16                            # al cl in parts that stay below 2^63
            first = al * (cl & 0xFFFF)
            carry = ((middle & low) + (first & low)) >> 32
            bottom = ((middle & low) + (first & low)) & low
            top = ((al * (cl >> 16)) >> 16) + (first >> 32) + carry
            return (top + al * (ch & 0xFFFF) + (((al * (ch >> 16)) & 0xFFFF) << 16) + ah * (cl & 0xFFFF)
                    + (((ah * (cl >> 16)) & 0xFFFF) << 16)) & low, bottom

        def shifted(a, n):  # a ^ a >> n, n below 32
            h, l = a
            return h ^ (h >> n), l ^ ((l >> n) | ((h << (32 - n)) & low))

        n = s["x"].numel()
        index = torch.arange((n + 1) // 2, dtype=torch.int64, device=s["x"].device)
        base = (SEED ^ STREAM * 0x9E3779B97F4A7C15 ^ int(s["tick"]) * 0xD1B54A32D192ED03) & ((1 << 64) - 1)
        h, l = times((index * 0, index), 0x94D049BB133111EB)
        v = shifted((h ^ (base >> 32), l ^ (base & low)), 30)
        v = shifted(times(v, 0xBF58476D1CE4E5B9), 27)
        h, l = shifted(times(v, 0x94D049BB133111EB), 31)
        kept = torch.stack([l, h], 1).flatten()[:n].view(s["x"].shape) / 2.0 ** 32 >= round(RATE * 2.0 ** 32) / 2.0 ** 32
        y = torch.where(kept, s["x"].double() / (1.0 - RATE), 0.0)
        result = {"y": y if s["residual"] is None else y + s["residual"].double()}
        if kind == "dropout_train":
            result["x"] = torch.where(kept, s["grad"].double() / (1.0 - RATE), 0.0)
        return result

    def embed():
        known = s["tokens"] >= 0
        out = s["grad"].double() * 0
        out[known] = SCALE * s["table"].double()[s["tokens"][known]]
        if kind == "embed":
            return {"out": out}
        table = torch.zeros(s["table"].shape, dtype=torch.float64, device=out.device)
        table.index_put_((s["tokens"][known],), SCALE * s["grad"].double()[known], accumulate=True)
        return {"out": out, "table": table}

    def linear():
        """S <- decay S + k v^T, o = S^T q / sqrt(dk), one token after the other; the gradients by the same steps
        backwards from states kept every 64 tokens."""
        step = kind == "linear_step"

        def heads_first(a):
            return (a.unsqueeze(1) if step else a).double().movedim(2, 1).contiguous()

        q, k, v = (heads_first(s[n]) for n in ("q", "k", "v"))
        B, Hv, T, dv = v.shape
        H, dk = q.shape[1], q.shape[3]
        q, k = (a.repeat_interleave(Hv // H, dim=1) for a in (q, k))
        g = s["log_decay"].double()
        g = g[None, :, None].expand(B, Hv, T) if case["decay"] == "head" else heads_first(s["log_decay"])
        live = torch.ones(B, T, dtype=torch.float64, device=v.device)
        if s.get("lengths") is not None:
            live = (torch.arange(T, device=v.device) < s["lengths"][:, None]).double()
        live = live[:, None, :]
        decay, k = torch.exp(g * live), k * live[..., None]
        scale = dk ** -0.5

        def advance(S, t):
            return S * decay[:, :, t, None, None] + k[:, :, t, :, None] * v[:, :, t, None, :]

        S = s["state"].double() if s.get("state") is not None else v.new_zeros(B, Hv, dk, dv)
        out, kept = torch.zeros_like(v), []
        for t in range(T):
            if t % 64 == 0:
                kept.append(S)
            S = advance(S, t)
            out[:, :, t] = scale * live[:, :, t, None] * (S * q[:, :, t, :, None]).sum(2)
        if step:
            return {"out": out[:, :, 0], "state": S}
        result = {"out": out.movedim(1, 2), "state": S}
        if "grad" not in s:
            return result
        do, dS = heads_first(s["grad"]) * live[..., None] * scale, s["grad_state"].double()
        dq, dk_, dv_, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(decay)
        for n in reversed(range(len(kept))):
            span, states = range(64 * n, min(T, 64 * n + 64)), [kept[n]]
            for t in span:
                states.append(advance(states[-1], t))
            for t in reversed(span):
                before, after = states[t - 64 * n], states[t - 64 * n + 1]
                dS = dS + q[:, :, t, :, None] * do[:, :, t, None, :]
                dq[:, :, t] = (after * do[:, :, t, None, :]).sum(3)
                dk_[:, :, t] = (dS * v[:, :, t, None, :]).sum(3)
                dv_[:, :, t] = (dS * k[:, :, t, :, None]).sum(2)
                dS = dS * decay[:, :, t, None, None]
                dg[:, :, t] = (dS * before).sum((2, 3))
        share = lambda a: a.reshape(B, H, Hv // H, T, dk).sum(2)  # noqa: E731
        grads = {"q": share(dq), "k": share(dk_ * live[..., None]), "v": dv_, "log_decay": dg * live}
        result.update({"grad_" + n: a.movedim(1, 2) for n, a in grads.items()})
        if case["decay"] == "head":
            result["grad_log_decay"] = (dg * live).sum((0, 2))
        if s.get("state") is not None:
            result["grad_state"] = dS
        return result

    return rms() if kind.startswith("rms") else dropout() if kind.startswith("dropout") else embed() if kind.startswith("embed") else linear()
