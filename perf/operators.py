"""The operators of ``atlas_hip.ops`` as measurable cases: layer normalisation of a layer's currents, the
gated delta rule (a fast-weight layer whose synapses decay and learn within a sequence) and the
orthogonalised weight update (Muon) that trains the dense matrices around them.

Sizes come from the recurrent trainer's plan (700 inputs -> 256 hidden -> 20 classes, 100 ticks, batch
256) or are generic.  ``run`` computes each operator in a plain form of elementary torch operations in
float32, rounded once at the end; with ``own`` set it calls the framework.  ``exact`` is the same from the
operators' definitions in float64: the delta rule token by token, its gradients by the reversed recurrence.
"""
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5                                   # layer normalisation
COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # the quintic iteration of the orthogonalisation
STEPS, NORM_EPS = 5, 1e-7
RATE, FACTOR, WEIGHT_DECAY = 0.02, 0.95, 0.01
CHUNK = 64                                   # tokens per chunk of the plain delta rule


def listed():
    return [
        # one tick's currents of the trainer's batch, normalised before the layer: launch latency counts
        {"name": "norm_tick", "kind": "norm", "rows": 256, "width": 256, "type": "f32"},
        # the same currents of a whole batch, 100 ticks of 256 samples: forward and backward
        {"name": "norm_train_ticks", "kind": "norm_train", "rows": 25600, "width": 256, "type": "f32"},
        # odd rows of an odd width: no vector access is aligned
        {"name": "norm_train_odd", "kind": "norm_train", "rows": 9973, "width": 1023, "type": "bf16"},
        # a wide layer over a large batch: memory bandwidth
        {"name": "norm_train_wide", "kind": "norm_train", "rows": 32768, "width": 4096, "type": "bf16"},
        # the trainer's recurrent matrix: a whole optimiser step, latency of a chain of small products
        {"name": "muon_recurrent", "kind": "muon", "batch": 1, "rows": 256, "columns": 256, "type": "f32"},
        # the matrices of several layers at once, of a ragged shape
        {"name": "orthogonalize_ragged", "kind": "orthogonalize", "batch": 6, "rows": 333, "columns": 1000,
         "type": "bf16"},
        # a large layer's matrix, taller than wide: matrix products
        {"name": "muon_large", "kind": "muon", "batch": 1, "rows": 4096, "columns": 2048, "type": "f32"},
        # streaming: one tick of 64 streams, a state of 128 x 128 for each of 8 heads
        {"name": "delta_tick", "kind": "delta_step", "batch": 64, "heads": 8, "value_heads": 8, "key": 128, "value": 128,
         "type": "bf16"},
        # the trainer's batch and ticks through 256 units as 4 heads of 64: forward and backward
        {"name": "delta_train_ticks", "kind": "delta_train", "batch": 256, "time": 100, "heads": 4, "value_heads": 4,
         "key": 64, "value": 64, "type": "f32", "ragged": False, "state": False},
        # one long recording through a wide layer: few rows, a long chain
        {"name": "delta_long", "kind": "delta", "batch": 1, "time": 16384, "heads": 16, "value_heads": 16, "key": 128,
         "value": 128, "type": "bf16", "ragged": False, "state": True},
        # training over long recordings that end at different ticks, keys shared by four value heads
        {"name": "delta_train_shared", "kind": "delta_train", "batch": 2, "time": 4099, "heads": 4, "value_heads": 16,
         "key": 128, "value": 128, "type": "bf16", "ragged": True, "state": True},
        # head widths that fill no tile, a few hundred ticks, ends inside a chunk
        {"name": "delta_train_odd", "kind": "delta_train", "batch": 3, "time": 777, "heads": 5, "value_heads": 5,
         "key": 48, "value": 72, "type": "f32", "ragged": True, "state": True},
    ]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    kind = rng.choice(["norm", "norm_train", "muon", "orthogonalize", "delta_step", "delta", "delta_train"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("norm", "norm_train"):
        width = spread(20, 8192)
        return {"kind": kind, "rows": spread(1, min(65536, (1 << 26) // width)), "width": width, "type": dtype}
    if kind in ("muon", "orthogonalize"):
        rows, columns = spread(16, 2048), spread(16, 2048)
        most = max(1, min(8, (1 << 22) // (rows * columns)))
        return {"kind": kind, "batch": spread(1, most), "rows": rows, "columns": columns, "type": dtype}
    heads = spread(1, 8)
    case = {"kind": kind, "batch": 0, "heads": heads, "value_heads": heads * rng.choice([1, 1, 2, 4]),
            "key": rng.choice([16, 32, 40, 64, 96, 128, spread(8, 128)]),
            "value": rng.choice([16, 32, 64, 96, 128, spread(8, 128)]), "type": dtype}
    if kind == "delta_step":
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
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=random, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=random, device=device)

    state = {"case": case}
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        rows, width = case["rows"], case["width"]
        # currents: units of their own mean and size, a sample's drive common to its units
        x = normal(rows, width) * (0.5 + uniform(width)) + 0.3 * normal(width) + 0.5 * normal(rows, 1)
        state["x"] = x.to(dtype)
        state["weight"] = 1.0 + 0.1 * normal(width)
        state["bias"] = 0.1 * normal(width)
        if kind == "norm_train":
            state["grad"] = normal(rows, width).to(dtype)
    elif kind in ("muon", "orthogonalize"):
        batch, rows, columns = case["batch"], case["rows"], case["columns"]
        # a weight gradient: a sum of outer products of a few strong directions over the noise of a batch
        rank = max(1, min(rows, columns) // 8)
        strength = torch.exp(-3.0 * torch.arange(rank, device=device) / rank)
        strong = torch.matmul(normal(batch, rows, rank) * strength, normal(batch, rank, columns)) / math.sqrt(rank)
        gradient = 1e-3 * (strong + normal(batch, rows, columns))
        if kind == "muon":
            gradient, shape = gradient.squeeze(0), (rows, columns) if batch == 1 else (batch, rows, columns)
            state["gradient"] = gradient.to(dtype)
            state["weight"] = normal(*shape) / math.sqrt(rows)
            state["momentum"] = 5e-3 * normal(*shape)
        else:
            state["matrix"] = gradient.to(dtype)
    else:
        B, H, Hv, dk, dv = case["batch"], case["heads"], case["value_heads"], case["key"], case["value"]
        lead = (B,) if kind == "delta_step" else (B, case["time"])
        # keys and queries of unit length, half of them along a common direction as firing rates are
        common = normal(dk).abs()
        q, k = (normal(*lead, H, dk) + 0.5 * common for _ in range(2))
        state["q"], state["k"] = ((a / a.norm(dim=-1, keepdim=True)).to(dtype) for a in (q, k))
        state["v"] = normal(*lead, Hv, dv).to(dtype)
        # decays from a few ticks to thousands, learning rates in (0, 1)
        state["log_decay"] = -torch.exp(-7.0 + 6.0 * uniform(*lead, Hv))
        state["beta"] = torch.sigmoid(normal(*lead, Hv))
        if kind == "delta_step" or case["state"]:
            state["state"] = 0.3 * normal(B, Hv, dk, dv)
        if kind != "delta_step":
            state["lengths"] = None
            if case["ragged"]:
                state["lengths"] = torch.randint(0, case["time"] + 1, (B,), generator=random, device=device,
                                                 dtype=torch.int32)
                state["lengths"][0] = case["time"]
        if kind == "delta_train":
            state["grad"] = normal(*lead, Hv, dv).to(dtype)
            state["grad_state"] = 0.1 * normal(B, Hv, dk, dv)
    return state


# ------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + EPS)
    normed = centred * rstd
    y = (normed * s["weight"] + s["bias"]).to(s["x"].dtype)
    if "grad" not in s:
        return {"y": y}
    grad = s["grad"].float()
    scaled = grad * s["weight"]
    dx = rstd * (scaled - scaled.mean(dim=-1, keepdim=True) - normed * (scaled * normed).mean(dim=-1, keepdim=True))
    return {"y": y, "x": dx.to(s["x"].dtype), "weight": (grad * normed).sum(dim=0), "bias": grad.sum(dim=0)}


def _orthogonal(x):
    a, b, c = COEFFICIENTS
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NORM_EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-2, -1).contiguous() if tall else x


def _plain_muon(s):
    weight, momentum, gradient = s["weight"], s["momentum"], s["gradient"].float()
    momentum.mul_(FACTOR).add_(gradient)
    update = _orthogonal(gradient + FACTOR * momentum)
    scale = math.sqrt(max(1.0, weight.shape[-1] / weight.shape[-2]))
    weight.mul_(1.0 - RATE * WEIGHT_DECAY).sub_(RATE * scale * update)
    return {"weight": weight, "momentum": momentum}


def _plain_delta_step(s):
    group = s["v"].shape[1] // s["q"].shape[1]
    q, k = (s[n].float().repeat_interleave(group, dim=1) for n in ("q", "k"))
    v, state = s["v"].float(), s["state"]
    scale = 1.0 / math.sqrt(q.shape[-1])
    state.mul_(torch.exp(s["log_decay"])[..., None, None])
    error = s["beta"][..., None] * (v - torch.matmul(k[..., None, :], state)[..., 0, :])
    state.add_(k[..., :, None] * error[..., None, :])
    return {"out": (scale * torch.matmul(q[..., None, :], state)[..., 0, :]).to(s["v"].dtype), "state": state}


def _chunked_delta(q, k, v, log_decay, beta, state, lengths):
    """Chunks of CHUNK tokens: within a chunk the corrections e solve (I + L) e = beta (v - decayed k S),
    L the decayed products of keys below the diagonal; the state is carried from chunk to chunk."""
    B, T, Hv, dv = v.shape
    group, dk = Hv // q.shape[2], q.shape[3]
    if lengths is not None:
        live = (torch.arange(T, device=v.device) < lengths[:, None]).float()[..., None]
        log_decay, beta = log_decay * live, beta * live
    chunks = -(-T // CHUNK)
    pad = chunks * CHUNK - T

    def split(a):  # (batch, time, heads, ...) -> (batch, heads, chunks, CHUNK, ...)
        a = torch.cat([a, a.new_zeros(B, pad, *a.shape[2:])], dim=1) if pad else a
        return a.reshape(B, chunks, CHUNK, *a.shape[2:]).movedim(3, 1).contiguous()

    q, k, v, g, beta = split(q), split(k), split(v), split(log_decay), split(beta)[..., None]
    q, k = (a.repeat_interleave(group, dim=1) for a in (q, k))
    g = g.cumsum(dim=-1)
    index = torch.arange(CHUNK, device=v.device)
    below = index[:, None] >= index
    decay = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~below, -math.inf))
    lower = beta * decay * torch.matmul(k, k.transpose(-2, -1)) * (index[:, None] > index)
    inverse = torch.eye(CHUNK, device=v.device).expand_as(lower)
    size = 1
    while size < CHUNK:  # the inverse of pairs of diagonal blocks from the inverses of the blocks
        row, column = index[:, None] // size, index // size
        pair = (row == column + 1) & (row % 2 == 1)
        inverse = inverse - torch.matmul(torch.matmul(inverse, lower * pair), inverse)
        size *= 2
    since = torch.exp(g)[..., None]
    rest = torch.exp(g[..., -1:] - g)[..., None]
    values, keys = torch.matmul(inverse, beta * v), torch.matmul(inverse, beta * since * k)
    queries = since * q / math.sqrt(dk)
    scores = decay * torch.matmul(q, k.transpose(-2, -1)) / math.sqrt(dk)
    writes = (rest * k).transpose(-2, -1)
    state = v.new_zeros(B, Hv, dk, dv) if state is None else state
    out = []
    for n in range(chunks):
        error = values[:, :, n] - torch.matmul(keys[:, :, n], state)
        out.append(torch.matmul(queries[:, :, n], state) + torch.matmul(scores[:, :, n], error))
        state = since[:, :, n, -1:] * state + torch.matmul(writes[:, :, n], error)
    out = torch.stack(out, dim=2).movedim(1, 3).reshape(B, chunks * CHUNK, Hv, dv)[:, :T]
    return out if lengths is None else out * live[..., None], state


def _plain_delta(s):
    train = "grad" in s
    names = ["q", "k", "v", "log_decay", "beta"] + (["state"] if "state" in s else [])
    leaves = {n: s[n].float().detach().requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        out, state = _chunked_delta(*(leaves.get(n) for n in ("q", "k", "v", "log_decay", "beta", "state")), s["lengths"])
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
    if kind == "norm":
        return {"y": ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)}
    if kind == "norm_train":
        y, mean, rstd = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, statistics=True)
        dx, dw, db = ops.layer_norm_backward(s["grad"], s["x"], s["weight"], mean, rstd)
        return {"y": y, "x": dx, "weight": dw, "bias": db}
    if kind == "muon":
        ops.muon_update(s["weight"], s["gradient"], s["momentum"], learning_rate=RATE, factor=FACTOR,
                        weight_decay=WEIGHT_DECAY)
        return {"weight": s["weight"], "momentum": s["momentum"]}
    if kind == "orthogonalize":
        return {"matrix": ops.orthogonalize(s["matrix"])}
    inputs = [s[n] for n in ("q", "k", "v", "log_decay", "beta")]
    if kind == "delta_step":
        return {"out": ops.delta_rule_step(*inputs, s["state"]), "state": s["state"]}
    if kind == "delta":
        out, state = ops.delta_rule(*inputs, s.get("state"), lengths=s["lengths"])
        return {"out": out, "state": state}
    out, state, tape = ops.delta_rule(*inputs, s.get("state"), lengths=s["lengths"], tape=True)
    grads = ops.delta_rule_backward(s["grad"], s["grad_state"], tape)
    result = {"out": out, "state": state}
    result.update({"grad_" + n: g for n, g in grads.items() if g is not None})
    return result


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("norm", "norm_train"):
        return _plain_norm(state)
    if kind == "muon":
        return _plain_muon(state)
    if kind == "orthogonalize":
        return {"matrix": _orthogonal(state["matrix"].float()).to(state["matrix"].dtype)}
    return _plain_delta_step(state) if kind == "delta_step" else _plain_delta(state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        n, w = case["rows"] * case["width"], case["width"]
        if kind == "norm":
            return {"bytes": 2 * n * size + 8 * w, "flops": 8 * n}
        return {"bytes": 4 * n * size + 16 * w, "flops": 20 * n}
    if kind in ("muon", "orthogonalize"):
        m, n = sorted((case["rows"], case["columns"]))
        values = case["batch"] * m * n
        # the two symmetric products need one triangle each
        flops = case["batch"] * STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        return {"bytes": values * (size + 16 if kind == "muon" else 2 * size), "flops": flops}
    tokens, Hv = case["batch"] * case.get("time", 1), case["value_heads"]
    qk, v = tokens * case["heads"] * case["key"], tokens * Hv * case["value"]
    cells = case["batch"] * Hv * case["key"] * case["value"]
    if kind == "delta_step":
        return {"bytes": size * (2 * qk + 2 * v) + 8 * tokens * Hv + 8 * cells, "flops": 6 * cells}
    given = 4 * cells * (2 if case["state"] else 1)
    if kind == "delta":
        return {"bytes": size * (2 * qk + 2 * v) + 8 * tokens * Hv + given,
                "flops": 6 * tokens * Hv * case["key"] * case["value"]}
    return {"bytes": size * (4 * qk + 4 * v) + 16 * tokens * Hv + 2 * given,
            "flops": 18 * tokens * Hv * case["key"] * case["value"]}


# -------------------------------------------------------------------------------- exact, in 64 bits
def _exact_norm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    variance, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sigma = torch.sqrt(variance + EPS)
    z = (x - mean) / sigma
    result = {"y": w * z + b}
    if "grad" in s:
        g = s["grad"].double()
        h = g * w
        result["x"] = (h - h.mean(1, keepdim=True) - z * (h * z).mean(1, keepdim=True)) / sigma
        result["weight"], result["bias"] = (g * z).sum(0), g.sum(0)
    return result


def _exact_orthogonal(x):
    a, b, c = COEFFICIENTS
    x = x / (torch.linalg.norm(x, dim=(-2, -1), keepdim=True) + NORM_EPS)
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT.contiguous()
            x = a * x + (b * g + c * (g @ g)) @ x
        else:
            g = x.mT.contiguous() @ x
            x = a * x + x @ (b * g + c * (g @ g))
    return x


def _exact_delta(s):
    """S <- decay S; e = v - S^T k; S <- S + beta k e^T; o = S^T q / sqrt(dk), one token after the other; the
    gradients by the same steps backwards from states kept every 64 tokens."""
    def heads_first(a):
        return a.double().movedim(2, 1).contiguous()

    q, k, v, g, beta = (heads_first(s[n]) for n in ("q", "k", "v", "log_decay", "beta"))
    B, Hv, T, dv = v.shape
    H, dk = q.shape[1], q.shape[3]
    q, k = (a.repeat_interleave(Hv // H, dim=1) for a in (q, k))
    live = torch.ones(B, T, dtype=torch.float64, device=v.device)
    if s.get("lengths") is not None:
        live = (torch.arange(T, device=v.device) < s["lengths"][:, None]).double()
    live = live[:, None, :]
    decay, beta = torch.exp(g * live), beta * live
    scale = dk ** -0.5

    def advance(S, t):
        S = S * decay[:, :, t, None, None]
        e = v[:, :, t] - (S * k[:, :, t, :, None]).sum(2)
        return S, e, S + (beta[:, :, t, None] * k[:, :, t])[..., None] * e[:, :, None, :]

    S = s["state"].double() if s.get("state") is not None else v.new_zeros(B, Hv, dk, dv)
    out, kept = torch.zeros_like(v), []
    for t in range(T):
        if t % 64 == 0:
            kept.append(S)
        _, _, S = advance(S, t)
        out[:, :, t] = scale * live[:, :, t, None] * (S * q[:, :, t, :, None]).sum(2)
    result = {"out": out.movedim(1, 2), "state": S}
    if "grad" not in s:
        return result
    do, dS = heads_first(s["grad"]) * live[..., None] * scale, s["grad_state"].double()
    dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, dbeta = torch.zeros_like(g), torch.zeros_like(g)
    for n in reversed(range(len(kept))):
        span, states = range(64 * n, min(T, 64 * n + 64)), [kept[n]]
        for t in span:
            states.append(advance(states[-1], t)[2])
        for t in reversed(span):
            before, after = states[t - 64 * n], states[t - 64 * n + 1]
            faded, e, _ = advance(before, t)
            kt, bt = k[:, :, t], beta[:, :, t, None]
            dS = dS + q[:, :, t, :, None] * do[:, :, t, None, :]
            dq[:, :, t] = (after * do[:, :, t, None, :]).sum(3)
            seen, back = (dS * e[:, :, None, :]).sum(3), (dS * kt[..., None]).sum(2)
            dbeta[:, :, t] = (kt * seen).sum(2)
            de = bt * back
            dv_[:, :, t] = de
            dk_[:, :, t] = bt * seen - (faded * de[:, :, None, :]).sum(3)
            dS = dS - kt[..., None] * de[:, :, None, :]
            dg[:, :, t] = (dS * faded).sum((2, 3))
            dS = dS * decay[:, :, t, None, None]
    share = lambda a: a.reshape(B, H, Hv // H, T, dk).sum(2)  # noqa: E731
    grads = {"q": share(dq), "k": share(dk_), "v": dv_, "log_decay": dg * live, "beta": dbeta * live}
    result.update({"grad_" + n: a.movedim(1, 2) for n, a in grads.items()})
    if s.get("state") is not None:
        result["grad_state"] = dS
    return result


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        return _exact_norm(s)
    if kind == "orthogonalize":
        return {"matrix": _exact_orthogonal(s["matrix"].double())}
    if kind == "muon":
        momentum = FACTOR * s["momentum"].double() + s["gradient"].double()
        update = _exact_orthogonal(s["gradient"].double() + FACTOR * momentum)
        scale = max(1.0, case["columns"] / case["rows"]) ** 0.5
        return {"weight": (1.0 - RATE * WEIGHT_DECAY) * s["weight"].double() - RATE * scale * update,
                "momentum": momentum}
    if kind == "delta_step":
        one = {n: s[n].unsqueeze(1) for n in ("q", "k", "v", "log_decay", "beta")}
        result = _exact_delta({**one, "state": s["state"]})
        return {"out": result["out"][:, 0], "state": result["state"]}
    return _exact_delta(s)
