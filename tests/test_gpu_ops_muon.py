"""The orthogonalised update on the GPU against the float64 reference (oracle/ops_oracle.py), which takes
it through the singular values.

Tolerances.  Rounding the iterates to 22 bits (and float32 sums) perturbs X by about 2^-23 |X|_F spread
over all directions at each of the steps; a perturbation of a weak direction grows by up to 3.4 a step,
485 over five, relative to its own start at |X|_F / sqrt(m).  The sum of the steps' perturbations grown to
the end, 2^-23 (1 + 3.4 + ... + 3.4^5) = 8.2e-5 of |X_0|_F = 1, is a bound on the error's Frobenius norm where
every direction is weak throughout; results have Frobenius norm sqrt(m), so 1e-4 sqrt(rank) bounds the
error of low-rank matrices too.  Matrices of full rank whose singular values reach one are held to 2e-5
of the result's norm.  bfloat16 results: half an ulp, 2^-9, on top.
"""
import math

import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def numpy(t):
    return t.double().cpu().numpy()


def make(shape, dtype=F32, seed=0, scale=1.0):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def error(got, want):
    return float(np.linalg.norm(numpy(got) - want) / np.linalg.norm(want))


SHAPES = [(1, 1), (1, 50), (50, 1), (16, 16), (20, 256), (256, 20), (63, 65), (64, 64), (65, 130), (129, 127), (256, 256),
          (700, 256), (333, 1000), (3, 40, 70), (5, 70, 40), (2, 1, 1), (130, 128, 9)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_matches_the_reference(shape, dtype):
    print(f"case: orthogonalize {shape} {dtype}", flush=True)
    m = make(shape, dtype, seed=sum(shape), scale=3e-3)
    got = ops.orthogonalize(m)
    assert got.dtype == dtype and got.shape == m.shape
    assert error(got, oo.orthogonalize(numpy(m))) <= 2e-5 + (2 ** -8 if dtype == BF16 else 0)
    assert torch.equal(got, ops.orthogonalize(m))


@pytest.mark.parametrize("shape", [(1990, 2050), (2050, 1990), (1990, 4100), (4100, 1990), (9, 700, 1300)])
def test_large_tiles(shape):
    """Sizes of the 64-tiles and of the 256 x 128 ones with split sums, ragged, both orientations, in a batch."""
    print(f"case: orthogonalize large {shape}", flush=True)
    m = make(shape, seed=4)
    got = ops.orthogonalize(m)
    x = m.double()
    a, b, c = ops.COEFFICIENTS
    x = x / (torch.linalg.norm(x, dim=(-2, -1), keepdim=True) + 1e-7)
    for _ in range(5):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT.contiguous()
            x = a * x + (b * g + c * (g @ g)) @ x
        else:
            g = x.mT.contiguous() @ x
            x = a * x + x @ (b * g + c * (g @ g))
    assert float((got.double() - x).norm() / x.norm()) <= 2e-5
    assert torch.equal(got, ops.orthogonalize(m))


@pytest.mark.parametrize("rank", [1, 4])
def test_low_rank(rank):
    print(f"case: orthogonalize rank {rank}", flush=True)
    m = make((200, rank), seed=1) @ make((rank, 300), seed=2)
    got, want = ops.orthogonalize(m), oo.orthogonalize(numpy(m))
    # the float32 input has a rounding noise of its own, which the iteration raises: part of the input
    assert np.linalg.norm(numpy(got) - want) <= 1e-4 * math.sqrt(rank) * 10


def test_a_wide_range_of_magnitudes():
    """Norms that overflow or vanish in a float32 sum of squares, and singular values over six decades."""
    print("case: orthogonalize magnitudes", flush=True)
    m = make((48, 80))
    want = oo.orthogonalize(numpy(m), eps=0.0)
    for scale in (1e30, 1e-30, 2.0 ** 120):
        got = ops.orthogonalize(m * scale, eps=0.0)
        assert error(got, oo.orthogonalize(numpy(m * scale), eps=0.0)) <= 2e-5
        assert error(got, want) <= 1e-4
    decades = m * torch.logspace(0, -6, 48, device="cuda")[:, None]
    want = oo.orthogonalize(numpy(decades))
    # against the largest term, as weak directions stay weak
    assert np.abs(numpy(ops.orthogonalize(decades)) - want).max() <= 2e-4


def test_steps_coefficients_and_special_values():
    print("case: orthogonalize options", flush=True)
    m = make((60, 90), seed=3)
    for steps, coefficients in ((1, ops.COEFFICIENTS), (3, (2.0, -1.5, 0.5)), (12, (1.875, -1.25, 0.375))):
        got = ops.orthogonalize(m, steps=steps, coefficients=coefficients)
        assert error(got, oo.orthogonalize(numpy(m), steps=steps, coefficients=coefficients)) <= 2e-5
    assert (ops.orthogonalize(torch.zeros(30, 40, device="cuda")) == 0).all()
    bad = make((2, 30, 40))
    bad[1, 3, 4] = float("nan")
    got = ops.orthogonalize(bad)
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all()
    assert ops.orthogonalize(torch.empty(0, 4, device="cuda")).shape == (0, 4)
    assert ops.orthogonalize(torch.empty(3, 0, 4, device="cuda")).shape == (3, 0, 4)


def test_strides():
    print("case: orthogonalize strides", flush=True)
    base = make((4, 60, 90))
    for view in (base[::2], base[:, 3:50:2, 5:77], base.transpose(0, 1), base.transpose(1, 2), base[1].T,
                 base[0:1].expand(3, 60, 90)):
        assert torch.equal(ops.orthogonalize(view), ops.orthogonalize(view.contiguous()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(256, 256), (700, 256), (256, 20), (3, 33, 47)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update_matches_the_reference(shape, dtype, nesterov):
    print(f"case: muon {shape} {dtype} {nesterov}", flush=True)
    weight, gradient, momentum = make(shape, seed=1), make(shape, dtype, seed=2), make(shape, seed=3)
    options = dict(learning_rate=0.05, factor=0.9, weight_decay=0.1, nesterov=nesterov)
    w, m = numpy(weight), numpy(momentum)
    for _ in range(3):
        w, m = oo.muon(w, numpy(gradient), m, **options)
        assert ops.muon_update(weight, gradient, momentum, **options) is None
    assert error(momentum, m) <= 2e-7          # three roundings of a sum of two terms
    assert error(weight, w) <= 1e-5            # three updates of at most 2e-5 each times the rate, and float32
    w, m = oo.muon(w, numpy(gradient), m, **options, scale=0.2)
    ops.muon_update(weight, gradient, momentum, **options, scale=0.2)
    assert error(weight, w) <= 1e-5


def test_update_bumps_versions_and_refuses():
    print("case: muon refusals", flush=True)
    w, g, m = make((30, 40)), make((30, 40), seed=1), make((30, 40), seed=2)
    before = w._version, m._version, g._version
    ops.muon_update(w, g, m, learning_rate=0.1)
    assert (w._version, m._version, g._version) == (before[0] + 1, before[1] + 1, before[2])
    for call in (lambda: ops.muon_update(w.T, g.T, m.T, learning_rate=0.1),
                 lambda: ops.muon_update(w, g[:29], m, learning_rate=0.1),
                 lambda: ops.muon_update(w, g, m.bfloat16(), learning_rate=0.1),
                 lambda: ops.muon_update(w.bfloat16(), g, m, learning_rate=0.1),
                 lambda: ops.muon_update(w, g.half(), m, learning_rate=0.1),
                 lambda: ops.muon_update(w, g, w, learning_rate=0.1), lambda: ops.muon_update(w, m, m, learning_rate=0.1),
                 lambda: ops.muon_update(w[0], g[0], m[0], learning_rate=0.1),
                 lambda: ops.muon_update(w, g, m, learning_rate=0.1, steps=0),
                 lambda: ops.orthogonalize(w, steps=65), lambda: ops.orthogonalize(w, coefficients=(1.0, 2.0)),
                 lambda: ops.orthogonalize(w.half()), lambda: ops.orthogonalize(w.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call()


def test_another_stream():
    print("case: muon stream", flush=True)
    m = make((300, 400))
    want = ops.orthogonalize(m)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.orthogonalize(m)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_sizes_beyond_the_limits_are_invalid_arguments():
    """Refused as such, and before anything is allocated for them."""
    print("case: muon limits", flush=True)
    one = torch.ones(1, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for shape in ((16385, 16385), (2, (1 << 20) + 1), ((1 << 20) + 1, 2), (65536, 1, 1)):
        with pytest.raises(ValueError, match="16384"):
            ops.orthogonalize(one.expand(shape))
    assert torch.cuda.max_memory_allocated() == before
    weight, momentum = torch.ones(65536, 1, 1, device="cuda"), torch.ones(65536, 1, 1, device="cuda")
    with pytest.raises(ValueError, match="16384"):
        ops.muon_update(weight, one.expand(65536, 1, 1), momentum, learning_rate=0.1)
    assert (weight == 1).all() and (momentum == 1).all()


def test_update_refuses_shared_memory():
    """Also where only a part is shared; a gradient whose gaps hold the others is taken."""
    print("case: muon shared memory", flush=True)
    flat = torch.randn(5000, generator=torch.Generator().manual_seed(8)).cuda()
    w, g, m = flat[:1200].view(30, 40), flat[1200:2400].view(30, 40), flat[2400:3600].view(30, 40)
    part = flat[100:1300].view(30, 40)
    halves = flat.bfloat16()
    for call in (lambda: ops.muon_update(w, g, part, learning_rate=0.1), lambda: ops.muon_update(w, part, m, learning_rate=0.1),
                 lambda: ops.muon_update(part, w.T.contiguous().T, w, learning_rate=0.1),
                 lambda: ops.muon_update(w, flat[2399:3599].view(30, 40), m, learning_rate=0.1),
                 lambda: ops.muon_update(w, flat[1100:2300].view(40, 30).T, m, learning_rate=0.1),
                 lambda: ops.muon_update(halves.view(F32)[:1200].view(30, 40), halves[2399:3599].view(30, 40), m, learning_rate=0.1)):
        with pytest.raises(ValueError, match="share memory"):
            call()
    wide = torch.randn(2, 2400, generator=torch.Generator().manual_seed(9)).cuda()
    gradient = wide[:, :600].unflatten(1, (20, 30))              # 2 x 20 x 30, with 1800 values between the two
    weight, momentum = wide[0, 600:1800].view(2, 20, 30), torch.zeros(2, 20, 30, device="cuda")
    alone, other, copy = weight.clone(), momentum.clone(), gradient.clone()
    ops.muon_update(alone, copy, other, learning_rate=0.1)
    ops.muon_update(weight, gradient, momentum, learning_rate=0.1)
    assert torch.equal(weight, alone) and torch.equal(momentum, other)


def test_coefficients_that_leave_the_range_are_refused():
    """Iterates lie in float16 planes, up to 4094: coefficients that raise any matrix's singular values, at most one at
    first, beyond that are refused, and those that stay below are held to 2e-5 of the result's norm; but where s grows
    as s^5, a rounding of 2^-22 grows five times a step, to 2^-22 (1 + 5 + ... + 5^6) = 4.7e-3 after six."""
    print("case: orthogonalize coefficients", flush=True)
    for m in (torch.ones(1, 1, device="cuda"), make((20, 30), seed=4), make((40, 1), seed=1) @ make((1, 50), seed=2)):
        for steps, coefficients, tol in ((2, (30.0, 0.0, 0.0), 2e-5), (1, (1e6, 0.0, 0.0), 2e-5), (1, (1.0, 2000.0, 1500.0), 2e-5),
                                         (64, (1.5, -0.5, 0.0), 2e-5), (20, ops.COEFFICIENTS, 2e-5), (6, (1e-3, 0.0, 1.0), 4.7e-3)):
            got, want = ops.orthogonalize(m, steps=steps, coefficients=coefficients), oo.orthogonalize(numpy(m), steps, coefficients)
            if min(m.shape) == 1 or m.shape[0] < m.shape[1] == 30:
                assert np.abs(numpy(got) - want).max() <= tol * max(1.0, np.linalg.norm(want)), (steps, coefficients)
            else:  # what the product's rounding leaves beside its rank grows by up to 3.4 a step: no exact value
                assert torch.isfinite(got).all()
        for steps, coefficients in ((3, (30.0, 0.0, 0.0)), (2, (5000.0, 0.0, 0.0)), (1, (1.0, 2500.0, 2000.0)),
                                    (9, (-2.0, -1.0, 0.0)), (5, (float("nan"), 0.0, 0.0)), (5, (1.0, 0.0, float("inf")))):
            with pytest.raises(ValueError, match="coefficients"):
                ops.orthogonalize(m, steps=steps, coefficients=coefficients)
            weight, momentum = torch.ones_like(m), torch.ones_like(m)
            with pytest.raises(ValueError, match="coefficients"):
                ops.muon_update(weight, m, momentum, learning_rate=0.1, steps=steps, coefficients=coefficients)
            assert (weight == 1).all() and (momentum == 1).all()


@pytest.mark.parametrize("shape", [(2050, 4100), (4100, 1990), (700, 1300)])
def test_update_of_large_matrices(shape):
    """The weight written out of the tiles of 256 x 128, both orientations, ragged, and of those of 64 x 64."""
    print(f"case: muon large {shape}", flush=True)
    weight, gradient, momentum = make(shape, seed=1), make(shape, seed=2), make(shape, seed=3)
    options = dict(learning_rate=0.05, factor=0.9, weight_decay=0.1)
    next_momentum = 0.9 * momentum.double() + gradient.double()
    x = gradient.double() + 0.9 * next_momentum
    x = x / (torch.linalg.norm(x) + 1e-7)
    a, b, c = ops.COEFFICIENTS
    for _ in range(5):
        if shape[0] <= shape[1]:
            g = x @ x.T.contiguous()
            x = a * x + (b * g + c * (g @ g)) @ x
        else:
            g = x.T.contiguous() @ x
            x = a * x + x @ (b * g + c * (g @ g))
    rate = 0.05 * math.sqrt(max(1.0, shape[1] / shape[0]))
    want = (1.0 - 0.05 * 0.1) * weight.double() - rate * x
    start = weight.double()
    ops.muon_update(weight, gradient, momentum, **options)
    assert float((momentum.double() - next_momentum).norm() / next_momentum.norm()) <= 2e-7
    # the step taken, to 2e-5 of it, and the weight's own rounding
    bound = 2e-5 * float((want - start).norm()) + 2.0 ** -24 * float(want.norm())
    assert float((weight.double() - want).norm()) <= bound


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_update_with_gradients_of_other_strides(dtype):
    print(f"case: muon strides {dtype}", flush=True)
    base = make((4, 60, 90), dtype, seed=5)
    wide = make((130, 80), dtype, seed=6)
    for gradient in (base.transpose(0, 1), base[:, 3:50:2, 5:77], base.transpose(1, 2), base[1].T, base[0:1].expand(3, 60, 90),
                     wide[::2, 1:78], wide[5:6].expand(30, 80)):
        results = []
        for g in (gradient, gradient.contiguous()):
            weight, momentum = make(g.shape, seed=1), make(g.shape, seed=2)
            ops.muon_update(weight, g, momentum, learning_rate=0.1)
            results.append((weight, momentum))
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rank", [1, 4])
def test_exactly_low_rank(rank):
    """Factors of small whole numbers: their product is exact in float32, so nothing but the iteration's own rounding
    stands outside the rank, held to the bound above."""
    print(f"case: orthogonalize exact rank {rank}", flush=True)
    g = torch.Generator().manual_seed(7)
    left, right = (torch.randint(-7, 8, s, generator=g).float() for s in ((200, rank), (rank, 300)))
    m = (left @ right).cuda()
    got, want = ops.orthogonalize(m), oo.orthogonalize(numpy(m))
    assert np.linalg.norm(numpy(got) - want) <= 1e-4 * math.sqrt(rank)
