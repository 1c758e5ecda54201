"""What every operator's call refuses alike: tensors whose memory does not hold what they stand for, and tensors that
carry forward-mode derivatives."""
import pytest
import torch
from torch.autograd import forward_ad

from atlas_hip import ops

pytestmark = pytest.mark.gpu


def tensors():
    g = torch.Generator().manual_seed(0)
    return {"x": torch.randn(4, 32, generator=g).cuda(), "m": torch.randn(4, 32, generator=g).cuda(),
            "k": torch.randn(2, 5, 1, 8, generator=g).cuda(), "gate": -torch.rand(2, 5, 1, generator=g).cuda()}


def calls(change):
    """Each operator with one tensor replaced by change(tensor)."""
    t = tensors()
    x, m, k, gate = t["x"], t["m"], t["k"], t["gate"]
    state = torch.zeros(2, 1, 8, 8, device="cuda")
    _, mean, rstd = ops.layer_norm(x, statistics=True)
    out, _, tape = ops.delta_rule(k, k, k, gate, -gate, tape=True)
    return {"layer_norm": lambda: ops.layer_norm(change(x)),
            "layer_norm weight": lambda: ops.layer_norm(x, change(x[0].clone())),
            "layer_norm_backward": lambda: ops.layer_norm_backward(change(m), x, None, mean, rstd),
            "orthogonalize": lambda: ops.orthogonalize(change(x)),
            "muon_update": lambda: ops.muon_update(x.clone(), change(m), torch.zeros_like(x), learning_rate=0.1),
            "delta_rule": lambda: ops.delta_rule(k, k, change(k), gate, -gate),
            "delta_rule gates": lambda: ops.delta_rule(k, k, k, change(gate), -gate),
            "delta_rule_step": lambda: ops.delta_rule_step(k[:, 0], k[:, 0], change(k[:, 0]), gate[:, 0], -gate[:, 0], state),
            "delta_rule_backward": lambda: ops.delta_rule_backward(change(out), None, tape)}


def test_tangents_are_refused():
    """A dual tensor's tangent would be dropped without a word."""
    print("case: dual tensors", flush=True)
    with forward_ad.dual_level():
        for name, call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))).items():
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls(lambda t: t).values():
            call()


def test_negated_views_are_refused():
    """Imaginary parts of conjugates are views that negate when they are read: their memory holds the other sign."""
    print("case: negated views", flush=True)
    def negated(t):
        view = torch.complex(t, -t).conj().imag
        assert view.is_neg() and torch.equal(view.resolve_neg(), t)
        return view

    for name, call in calls(negated).items():
        with pytest.raises(ValueError, match="resolve_neg"):
            call()


def test_what_is_no_tensor_is_refused():
    print("case: no tensors", flush=True)
    t = tensors()
    x, k, gate = t["x"], t["k"], t["gate"]
    _, mean, rstd = ops.layer_norm(x, statistics=True)
    out = ops.delta_rule(k, k, k, gate, -gate)[0]
    for call in (lambda: ops.layer_norm_backward(x, x, [1.0] * 32, mean, rstd), lambda: ops.layer_norm_backward(x, x, None, 0.0, 1.0),
                 lambda: ops.delta_rule(k, k, None, gate, -gate), lambda: ops.delta_rule(None, k, k, gate, -gate),
                 lambda: ops.delta_rule(k, k, k, gate, -gate, state=0.0), lambda: ops.delta_rule(k, k, k, gate, -gate, lengths=[1, 2]),
                 lambda: ops.delta_rule_backward(out, None, None), lambda: ops.delta_rule_backward(out, None, (out, out)),
                 lambda: ops.delta_rule_step(k[:, 0], k[:, 0], None, gate[:, 0], -gate[:, 0], torch.zeros(2, 1, 8, 8, device="cuda")),
                 lambda: ops.layer_norm(None), lambda: ops.orthogonalize([[1.0]]),
                 lambda: ops.muon_update(x, None, torch.zeros_like(x), learning_rate=0.1)):
        with pytest.raises(ValueError):
            call()
