"""Root-mean-square normalisation on the GPU against the float64 reference (oracle/ops_oracle.py).

Tolerances, in roundings of 2^-24.  A row's sum of squares adds at most width / 256 + 32 terms one after the other (a lane's
own, then lanes and waves by halves); every step from there to y and dx is a product or a sum of a few terms: UNITS(width)
= width / 256 + 48 of the size of the terms.  A column sum of g z adds a group's rows one after the other, then up to
16 groups, 768 / 32 workgroups and 32 parts.  A result of fewer bits is rounded once: bfloat16 2^-8 of its value, e4m3 half
its spacing there.
"""
import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ULP = 2.0 ** -24
ROUND = {F32: ULP, BF16: 2.0 ** -8}


def numpy(t):
    return t.double().cpu().numpy()


def make(shape, dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) + offset).to(dtype).cuda()


def close(got, want, scale, units, what):
    bound = units * ULP * scale + ROUND[got.dtype] * np.abs(want) + 1e-37
    error = np.abs(numpy(got) - want)
    assert (error <= bound).all(), (what, float((error / bound).max()))


def check(x, weight, residual, grad, grad_total=None, eps=1e-5):
    width = x.shape[-1]
    units = width / 256 + 48
    y, *rest = ops.rms_norm(x, weight, residual, eps=eps, statistics=True)
    rstd, total = rest[-1], x if residual is None else rest[0]
    if residual is not None:
        assert torch.equal(total, (x.float() + residual.float()).to(x.dtype)), "one rounding"
    w = None if weight is None else numpy(weight)
    want, wrstd = oo.rms_norm(numpy(total), w, eps)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == x.shape
    close(y, want, np.abs(want), units, "y")
    assert (np.abs(numpy(rstd) - wrstd) <= units * ULP * wrstd).all()
    without = ops.rms_norm(x, weight, residual, eps=eps)
    assert torch.equal(y, without if residual is None else without[0])
    dx, dw = ops.rms_norm_backward(grad, total, weight, rstd, grad_total=grad_total)
    s = None if grad_total is None else numpy(grad_total)
    gx, gw = oo.rms_norm_backward(numpy(grad), numpy(total), w, s, eps)
    h, z = np.abs(numpy(grad) * (1.0 if w is None else w)), np.abs(numpy(total)) * wrstd[..., None]
    terms = wrstd[..., None] * (h + z * (h * z).mean(axis=-1, keepdims=True)) + (0.0 if s is None else np.abs(s))
    close(dx, gx, terms, units, "dx")
    rows = x.numel() // width
    close(dw, gw, (np.abs(numpy(grad)) * z).reshape(-1, width).sum(axis=0), rows / 64 + 128 + units, "dweight")
    assert dw.dtype == (F32 if weight is None else weight.dtype)
    again = ops.rms_norm_backward(grad, total, weight, rstd, grad_total=grad_total)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]), "the same bits on every run"
    assert torch.equal(dx, ops.rms_norm_backward(grad, total, weight, rstd, grad_total=grad_total, sums=False)[0])
    check_8bit(x, weight, residual, total, want, eps, units)


def check_8bit(x, weight, residual, total, want, eps, units):
    values, scale, *rest = ops.rms_norm_8bit(x, weight, residual, eps=eps)
    assert values.dtype == torch.float8_e4m3fn and values.shape == x.shape and scale.shape == x.shape[:-1]
    assert len(rest) == (residual is not None) and (not rest or torch.equal(rest[0], total))
    most = np.maximum(np.abs(want).max(axis=-1) / 448.0, 2.0 ** -126)
    assert (np.abs(numpy(scale) - most) <= units * ULP * most).all()
    got, exact = numpy(values.float()), want / numpy(scale)[..., None]
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(exact), 2.0 ** -6))) - 3)
    error = np.abs(got - exact)
    assert (error <= step / 2 + units * ULP * np.abs(exact) * 2).all(), float((error / step).max())


# widths on both sides of every layout: a lane's 16 bytes, 16 lanes, a wave, a workgroup, beyond its registers
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (17, 20), (5, 64), (33, 65), (64, 128), (7, 129), (300, 256),
                                        (41, 257), (9, 513), (9, 700), (130, 1023), (12, 1024), (11, 1025), (5, 2048),
                                        (9, 2049), (3, 4097), (2, 8192), (70, 8193), (3, 20001)])
def test_matches_the_reference(rows, width, dtype):
    print(f"case: rms norm {rows} x {width} {dtype}", flush=True)
    x, grad = make((rows, width), dtype), make((rows, width), dtype, 1, 0.1)
    check(x, make(width, F32, 2, 1.0), make((rows, width), dtype, 3), grad, make((rows, width), dtype, 4, 0.0))
    check(x, make(width, F32, 2, 1.0), None, grad)


@pytest.mark.parametrize("dtype,wtype", [(F32, None), (BF16, None), (BF16, BF16), (BF16, F32)])
def test_weights_of_each_kind(dtype, wtype):
    print(f"case: rms norm weights {dtype} {wtype}", flush=True)
    x, grad = make((37, 192), dtype), make((37, 192), dtype, 1, 0.1)
    weight = None if wtype is None else make(192, wtype, 2, 1.0)
    check(x, weight, None, grad, make((37, 192), dtype, 5))
    check(x, weight, make((37, 192), dtype, 3), grad)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(33001, 20), (20001, 256), (9001, 300), (9001, 1000), (2000, 1500), (2600, 2000),
                                        (1700, 4000), (700, 6000), (150, 9000), (90, 17000)])
def test_several_rows_in_each_place(rows, width, dtype):
    """More rows than the grid has places for, all of them different, in every layout of a row."""
    print(f"case: rms norm rows {rows} x {width} {dtype}", flush=True)
    x, grad = make((rows, width), dtype, 4), make((rows, width), dtype, 5, 0.1)
    check(x, make(width, F32, 2, 1.0), make((rows, width), dtype, 6), grad, make((rows, width), dtype, 7))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    print(f"case: rms norm strides {dtype}", flush=True)
    base, add, grad, stream = (make((6, 5, 4, 40), dtype, seed) for seed in range(4))
    weight = make(80, F32, 2, 1.0)[::2]
    for view in (lambda t: t.transpose(0, 1), lambda t: t.permute(2, 1, 0, 3), lambda t: t[:, ::2], lambda t: t[1:, :, 1:3],
                 lambda t: t[0, 0, 0]):
        check(view(base), weight, view(add), view(grad), view(stream))
    # each of its own strides: an unaligned start, a broadcast residual, a last axis that is not contiguous
    flat = make(12 * 40 + 3, dtype)
    check(flat[3:].view(12, 40), weight, add[0, 0, 0].expand(12, 40), grad[0, 0, 0].expand(12, 40), stream[0].reshape(20, 40)[:12])
    check(base[:, 0].transpose(1, 2), None, add[:, 0].transpose(1, 2), grad[:, 0].transpose(1, 2).contiguous())


def test_special_values():
    print("case: rms norm special values", flush=True)
    x = make((7, 96), F32)
    x[1], x[6] = 0.0, 1e-30
    x[2, 5], x[3, 7], x[4, 0] = float("nan"), float("inf"), -float("inf")
    y, rstd = ops.rms_norm(x, statistics=True)
    assert (y[1] == 0).all() and torch.isfinite(y[[0, 1, 5, 6]]).all() and torch.isnan(y[2]).all()
    assert torch.isnan(y[3, 7]) and (y[3, :7] == 0).all(), "an infinite row is zero but where it is infinite"
    dx, _ = ops.rms_norm_backward(make((7, 96), F32, 1), x, None, rstd)
    assert torch.isfinite(dx[[0, 1, 5, 6]]).all() and torch.isnan(dx[2]).all()
    values, scale = ops.rms_norm_8bit(x)
    assert scale[1] == 2.0 ** -126 and (values[1].float() == 0).all() and torch.isnan(values[2].float()).all()
    weight = torch.ones(96, device="cuda")
    weight[3] = float("nan")
    values, scale = ops.rms_norm_8bit(x[:1], weight)
    assert torch.isfinite(scale).all() and torch.isnan(values[0, 3].float()) and torch.isfinite(values[0, 4:].float()).all()


def test_zero_gradient_rows_and_eps():
    """Rows of zeros have gradients of grad / sqrt(eps), as the formula says."""
    print("case: rms norm zero rows", flush=True)
    x, grad = torch.zeros(4, 64, device="cuda"), make((4, 64), F32, 1)
    _, rstd = ops.rms_norm(x, eps=1e-4, statistics=True)
    dx, dw = ops.rms_norm_backward(grad, x, None, rstd)
    assert (dx - grad * 100).abs().max() <= 1e-4 and (dw == 0).all()


def test_empty_and_refused():
    print("case: rms norm empty", flush=True)
    x, weight = torch.empty(0, 5, 32, device="cuda"), torch.ones(32, device="cuda")
    y, total, rstd = ops.rms_norm(x, weight, x, statistics=True)
    assert y.shape == total.shape == x.shape and rstd.shape == (0, 5)
    dx, dw = ops.rms_norm_backward(x, x, weight, rstd)
    assert dx.shape == x.shape and (dw == 0).all() and dw.shape == (32,)
    values, scale = ops.rms_norm_8bit(x)
    assert values.shape == x.shape and scale.shape == (0, 5)
    x = make((4, 32), F32)
    rstd = ops.rms_norm(x, statistics=True)[1]
    for call in (lambda: ops.rms_norm(x.half()), lambda: ops.rms_norm(x, weight[:31]), lambda: ops.rms_norm(x, weight.bfloat16()),
                 lambda: ops.rms_norm(x[:, :0]), lambda: ops.rms_norm(x, weight.cpu()), lambda: ops.rms_norm(x, None, x[:3]),
                 lambda: ops.rms_norm(x, None, x.bfloat16()), lambda: ops.rms_norm(x, None, x.cpu()), lambda: ops.rms_norm(None),
                 lambda: ops.rms_norm(x.clone().requires_grad_()), lambda: ops.rms_norm(torch.tensor(1.0).cuda()),
                 lambda: ops.rms_norm(x, None, 0.0), lambda: ops.rms_norm_8bit(x.half()), lambda: ops.rms_norm_8bit(x, None, x[:3]),
                 lambda: ops.rms_norm_backward(x.bfloat16(), x, None, rstd), lambda: ops.rms_norm_backward(x[:3], x, None, rstd),
                 lambda: ops.rms_norm_backward(x, x, None, rstd[:2]), lambda: ops.rms_norm_backward(x, x, None, rstd.double()),
                 lambda: ops.rms_norm_backward(x, x, None, rstd, grad_total=x[:2]),
                 lambda: ops.rms_norm_backward(x, x, None, rstd, grad_total=x.bfloat16())):
        with pytest.raises(ValueError):
            call()


def test_offsets_beyond_32_bits():
    """A result of 2^31 + values, and rows 2^31 elements apart."""
    print("case: rms norm offsets", flush=True)
    width, rows = 8192, (1 << 18) + 3
    row = make((1, width), BF16)
    many = row.expand(rows, width)
    y, total, rstd = ops.rms_norm(many, None, many, statistics=True)
    for t in (y, total):
        assert torch.equal(t[-1], t[0]) and torch.equal(t[rows // 2], t[0])
    dx, _ = ops.rms_norm_backward(many, total, None, rstd, grad_total=many)
    assert torch.equal(dx[-1], dx[0])
    del y, dx, total
    values, _ = ops.rms_norm_8bit(many)
    assert torch.equal(values[-1].float(), values[0].float())
    del values
    memory = torch.empty((1 << 31) + 64, dtype=BF16, device="cuda")
    far = memory.as_strided((2, 64), (1 << 31, 1))
    far.copy_(make((2, 64), BF16, 7))
    check(far, None, far, make((2, 64), BF16, 8), far)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [20, 96, 300, 1000, 1500, 4000, 9000])
def test_8bit_rows_beyond_float32(width, dtype):
    """Rows whose squares pass float32 have an infinite scale in every layout: an infinity of either sign, one that the residual
    brings, and finite values too large.  So has a row with an infinite weight; their neighbours keep theirs."""
    print(f"case: rms norm 8 bits beyond float32, {width} {dtype}", flush=True)
    x = make((6, width), dtype)
    clean = ops.rms_norm_8bit(x)
    dirty, residual = x.clone(), torch.zeros_like(x)
    dirty[1, width // 2], dirty[2, 0], residual[3, width - 1], dirty[4] = float("inf"), -float("inf"), float("inf"), 3e19
    values, scale, total = ops.rms_norm_8bit(dirty, None, residual)
    assert torch.isinf(scale[1:5]).all() and (scale[1:5] > 0).all()
    for row in (0, 5):
        assert scale[row] == clean[1][row] and torch.equal(values[row].float(), clean[0][row].float())
    assert torch.isnan(values[1, width // 2].float()) and torch.isnan(values[2, 0].float()) and torch.isnan(values[3, width - 1].float())
    assert (values[4].float() == 0).all() and (values[1].float() == 0).sum() == width - 1
    dirty = x.clone()
    dirty[1, 3] = float("nan")   # of a NaN no scale knows: the values are NaN
    values, scale = ops.rms_norm_8bit(dirty)
    assert torch.isnan(values[1].float()).all() and scale[1] == 2.0 ** -126
    weight = torch.ones(width, device="cuda")
    weight[5] = float("inf")
    values, scale = ops.rms_norm_8bit(x, weight)
    assert torch.isinf(scale).all()


@pytest.mark.parametrize("width", [(1 << 27) - 32, (1 << 27) + 40])
def test_column_sums_of_the_widest_rows(width):
    """On both sides of 2^27 columns, where a workgroup of 1024 threads for 32 columns would pass 2^32 threads."""
    print(f"case: rms norm column sums of {width}", flush=True)
    x = torch.ones(1, width, dtype=BF16, device="cuda")
    x[0, ::3] = 2.0
    y, rstd = ops.rms_norm(x, statistics=True)
    dx, dw = ops.rms_norm_backward(x, x, None, rstd)
    square = float((x[0, :3].double() ** 2).sum() / 3)
    assert abs(rstd.item() - square ** -0.5) <= 1e-3 * square ** -0.5
    want = x[0].float() * (x[0].float() * rstd[0])
    assert torch.equal(dw, want), "one row: the sum is its product"
