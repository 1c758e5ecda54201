"""Layer normalisation on the GPU against the float64 reference (oracle/ops_oracle.py).

Tolerances.  The kernels hold a row in float32: its mean and variance are sums of `width` terms by halves,
so their relative error is below (4 + log2 width) ulp, and z = (x - mean) rstd inherits the mean's error
amplified by |mean| / sigma.  With the inputs here (|mean| of the order of sigma) 32 ulp of the largest
term, 2^-19 = 2e-6, bounds y and dx.  The mean's error is an absolute one of z, of the order of an ulp of
one, also where z itself is small: a column sum of g z is off by up to 2e-6 of its sum of |g| (|z| + 1),
one of g by 2e-6 of its sum of |g|.  A bfloat16 result is rounded once: half an ulp, 2^-9 of the value, on top.
"""
import numpy as np
import pytest
import torch

from atlas_hip import ops
from oracle import ops_oracle as oo

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = 2e-6
ROUND = {F32: 0.0, BF16: 2.0 ** -8}   # a rounding that lands on the other side of a tie counts whole


def numpy(t):
    return t.double().cpu().numpy()


def make(shape, dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) + offset).to(dtype).cuda()


def close(got, want, scale, dtype, what):
    bound = TOL * scale + ROUND[dtype] * np.abs(want) + 1e-30
    error = np.abs(numpy(got) - want)
    assert got.dtype == dtype and (error <= bound).all(), (what, float((error / bound).max()))


def check(x, weight, bias, grad, eps=1e-5):
    y, mean, rstd = ops.layer_norm(x, weight, bias, eps=eps, statistics=True)
    w = None if weight is None else numpy(weight)
    want, wmean, wrstd = oo.layer_norm(numpy(x), w, None if bias is None else numpy(bias), eps)
    size = float(np.abs(want).max()) + (0.0 if bias is None else float(np.abs(numpy(bias)).max()))
    close(y, want, size, x.dtype, "y")
    assert torch.equal(y, ops.layer_norm(x, weight, bias, eps=eps))
    np.testing.assert_allclose(numpy(mean), wmean, rtol=0, atol=TOL * float(np.abs(numpy(x)).max()))
    np.testing.assert_allclose(numpy(rstd), wrstd, rtol=8 * TOL)
    dx, dw, db = ops.layer_norm_backward(grad, x, weight, mean, rstd)
    gx, gw, gb = oo.layer_norm_backward(numpy(grad), numpy(x), w, eps)
    close(dx, gx, float(np.abs(gx).max()) * 4 + float(np.abs(wrstd).max() * np.abs(numpy(grad)).max()), x.dtype, "dx")
    z = oo.layer_norm(numpy(x), eps=eps)[0]
    g = numpy(grad).reshape(-1, x.shape[-1])
    wtype = F32 if weight is None else weight.dtype
    close(dw, gw, (np.abs(g) * (np.abs(z.reshape(g.shape)) + 1.0)).sum(axis=0), wtype, "dweight")
    close(db, gb, np.abs(g).sum(axis=0) + 1e-6, wtype, "dbias")
    again = ops.layer_norm_backward(grad, x, weight, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again)), "the same bits on every run"


# widths on both sides of every layout: a lane's 16 bytes, 16 lanes, a wave, a workgroup, beyond its registers
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (17, 20), (5, 64), (33, 65), (64, 128), (7, 129), (300, 256),
                                        (41, 257), (9, 700), (130, 1023), (12, 1024), (11, 1025), (5, 2048),
                                        (9, 2049), (3, 4099), (2, 8192), (70, 8193), (3, 20001)])
def test_matches_the_reference(rows, width, dtype):
    print(f"case: layer norm {rows} x {width} {dtype}", flush=True)
    x, grad = make((rows, width), dtype), make((rows, width), dtype, 1, 0.1)
    check(x, make(width, F32, 2, 1.0), make(width, F32, 3, 0.0), grad)


@pytest.mark.parametrize("dtype,wtype", [(F32, None), (BF16, None), (BF16, BF16), (BF16, F32)])
def test_weights_of_each_kind(dtype, wtype):
    print(f"case: layer norm weights {dtype} {wtype}", flush=True)
    x, grad = make((37, 192), dtype), make((37, 192), dtype, 1, 0.1)
    weight = None if wtype is None else make(192, wtype, 2, 1.0)
    check(x, weight, None, grad)
    check(x, None if weight is None else weight, None if wtype is None else make(192, wtype, 3), grad)


def test_many_rows():
    print("case: layer norm 20000 x 256", flush=True)
    check(make((20000, 256), F32), make(256, F32, 2, 1.0), make(256, F32, 3), make((20000, 256), F32, 1, 0.1))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    print(f"case: layer norm strides {dtype}", flush=True)
    base = make((6, 5, 4, 40), dtype)
    grad = make((6, 5, 4, 40), dtype, 1, 0.1)
    weight, bias = make(80, F32, 2, 1.0)[::2], make(40, F32, 3)
    for view in (lambda t: t, lambda t: t.transpose(0, 1), lambda t: t.permute(2, 1, 0, 3), lambda t: t[:, ::2],
                 lambda t: t[1:, :, 1:3], lambda t: t[0, 0], lambda t: t[0, 0, 0]):
        x, g = view(base), view(grad)
        check(x, weight, bias, g)
    # an unaligned start, a last axis that is not contiguous, a broadcast gradient
    flat = make(12 * 40 + 3, dtype)
    check(flat[3:].view(12, 40), weight, bias, grad[0, 0, 0].expand(12, 40))
    check(base.transpose(2, 3)[..., :1, :].reshape(30, 4), None, None, grad.transpose(2, 3)[..., :1, :].reshape(30, 4))
    x = base[:, 0].transpose(1, 2)
    check(x, None, None, grad[:, 0].transpose(1, 2))


def test_a_large_mean_does_not_cancel():
    """Mean 4096 sigma: with E[x^2] - mean^2 the variance would be lost; of the centred squares it is not."""
    print("case: layer norm large mean", flush=True)
    x = torch.randn(8, 512, generator=torch.Generator().manual_seed(0)).double() + 4096.0
    x = x.float().cuda()
    y = ops.layer_norm(x)
    # mean's rounding, half an ulp of 4096, is 2.4e-4 of sigma
    np.testing.assert_allclose(numpy(y), oo.layer_norm(numpy(x))[0], rtol=0, atol=3e-4)


def test_special_values():
    print("case: layer norm special values", flush=True)
    x = make((6, 96), F32)
    x[1] = 3.0                     # no variance
    x[2, 5], x[3, 7], x[4, 0] = float("nan"), float("inf"), -float("inf")
    grad = make((6, 96), F32, 1)
    y, mean, rstd = ops.layer_norm(x, statistics=True)
    assert (y[1] == 0).all() and torch.isfinite(y[[0, 1, 5]]).all()
    assert torch.isnan(y[2:5]).all(dim=1).all()
    dx, _, _ = ops.layer_norm_backward(grad, x, None, mean, rstd)
    assert torch.isfinite(dx[[0, 1, 5]]).all() and torch.isnan(dx[2:5]).all()
    tiny = torch.full((2, 64), 1e-30, device="cuda")
    assert (ops.layer_norm(tiny) == 0).all()


def test_empty_and_refused():
    print("case: layer norm empty", flush=True)
    x = torch.empty(0, 5, 32, device="cuda")
    weight = torch.ones(32, device="cuda")
    y, mean, rstd = ops.layer_norm(x, weight, statistics=True)
    assert y.shape == x.shape and mean.shape == (0, 5)
    dx, dw, db = ops.layer_norm_backward(x, x, weight, mean, rstd)
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all() and dw.shape == (32,)
    x = make((4, 32), F32)
    mean, rstd = ops.layer_norm(x, statistics=True)[1:]
    for call in (lambda: ops.layer_norm(x.half()), lambda: ops.layer_norm(x, weight[:31]),
                 lambda: ops.layer_norm(x, weight.bfloat16()), lambda: ops.layer_norm(x[:, :0]),
                 lambda: ops.layer_norm(x, weight.cpu()), lambda: ops.layer_norm(x.bfloat16(), weight, weight.bfloat16()),
                 lambda: ops.layer_norm(x.clone().requires_grad_()), lambda: ops.layer_norm(torch.tensor(1.0).cuda()),
                 lambda: ops.layer_norm_backward(x.bfloat16(), x, None, mean, rstd),
                 lambda: ops.layer_norm_backward(x[:3], x, None, mean, rstd),
                 lambda: ops.layer_norm_backward(x, x, None, mean[:2], rstd),
                 lambda: ops.layer_norm_backward(x, x, None, mean, rstd.double())):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        ops.layer_norm(x.clone().requires_grad_())
    dx, dw, db = ops.layer_norm_backward(x, x, None, mean, rstd, sums=False)
    assert dw is None and db is None


def test_offsets_beyond_32_bits():
    """A result of 2^31 + values, and rows 2^31 elements apart."""
    print("case: layer norm offsets", flush=True)
    width, rows = 8192, (1 << 18) + 3
    row = make((1, width), BF16)
    y, mean, rstd = ops.layer_norm(row.expand(rows, width), statistics=True)
    assert torch.equal(y[-1], y[0]) and torch.equal(y[rows // 2], y[0])
    dx, dw, _ = ops.layer_norm_backward(row.expand(rows, width), row.expand(rows, width), None, mean, rstd)
    assert torch.equal(dx[-1], dx[0])
    del y, dx
    memory = torch.empty((1 << 31) + 64, dtype=BF16, device="cuda")
    far = memory.as_strided((2, 64), (1 << 31, 1))
    far.copy_(make((2, 64), BF16, 7))
    check(far, None, None, make((2, 64), BF16, 8))


def test_another_stream():
    print("case: layer norm stream", flush=True)
    x = make((512, 300), F32)
    want = ops.layer_norm(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.layer_norm(x)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(33001, 20), (26001, 48), (9001, 300), (6001, 500), (9001, 1000), (2000, 1500),
                                        (2600, 2000), (1700, 3000), (2200, 4000), (150, 6000), (150, 9000)])
def test_several_rows_in_each_place(rows, width, dtype):
    """More rows than the grid has places for, all of them different, in every layout of a row: the next row's fetch,
    the shared sums and the column sums go round."""
    print(f"case: layer norm rows {rows} x {width} {dtype}", flush=True)
    x, grad = make((rows, width), dtype, 4), make((rows, width), dtype, 5, 0.1)
    check(x, make(width, F32, 2, 1.0), make(width, F32, 3, 0.0), grad)


@pytest.mark.parametrize("width", [(1 << 26) - 16, (1 << 26) + 40])
def test_column_sums_of_the_widest_rows(width):
    """On both sides of 2^26 columns, where a workgroup of 1024 threads for 32 of both sums' columns would pass 2^32 threads."""
    print(f"case: layer norm column sums of {width}", flush=True)
    # half of the values 2, half 1: a mean of 1.5.  From there six roundings of 2^-24 of at most 2 x 2 x 2.
    x = torch.ones(1, width, dtype=BF16, device="cuda")
    x[0, ::2] = 2.0
    _, mean, rstd = ops.layer_norm(x, statistics=True)
    dx, dweight, dbias = ops.layer_norm_backward(x, x, None, mean, rstd)
    want = x[0].float() * ((x[0].float() - 1.5) * rstd[0])
    assert (dweight - want).abs().max() <= 48 * 2.0 ** -24 and torch.equal(dbias, x[0].float()), "one row: the sum is its product"
