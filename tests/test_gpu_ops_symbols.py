"""Embedding, its gradient and dropout on the GPU against the float64 reference (oracle/ops_oracle.py).

Tolerances.  A looked-up value is one product, rounded once: equal to the same product in float32, rounded to the table's
type.  A row of the gradient adds up to 32 values one after the other in a tile of 8 to 32 places, then the tiles' sums in up to
64 parts in order, and those: 32 + n / 512 + 64 for its n tokens.  Where one launch takes few symbols, 128 groups add n / 128
values each, and 3 + 16 sums join them.  Either is below 96 + n / 32 roundings of 2^-24 of the sum of magnitudes; one more for the
scale, and one to the table's type (bfloat16 2^-8).  Dropout keeps exactly what the reference keeps; a value is one product and, with a residual,
one sum: 2 roundings.
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


def make(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def check_gradient(grad, tokens, rows, scale=1.0, dtype=None):
    got = ops.embedding_backward(grad, tokens, rows, scale=scale, dtype=dtype)
    assert got.dtype == (dtype or grad.dtype) and got.shape == (rows, grad.shape[-1])
    flat = tokens.cpu().numpy().reshape(-1)
    want = oo.embedding_backward(numpy(grad), flat, rows, scale)
    size = oo.embedding_backward(np.abs(numpy(grad)), flat, rows, abs(scale))
    counts = np.bincount(flat[(flat >= 0) & (flat < rows)], minlength=rows)[:, None]
    bound = (97 + counts / 32) * ULP * size + ROUND[got.dtype] * np.abs(want)
    error = np.abs(numpy(got) - want)
    assert (error <= bound).all(), float((error / np.maximum(bound, 1e-300)).max())
    assert (numpy(got)[counts[:, 0] == 0] == 0).all()
    assert torch.equal(got, ops.embedding_backward(grad, tokens, rows, scale=scale, dtype=dtype)), "the same bits on every run"


def drawn(shape, rows, kind, seed=0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(shape, generator=g, dtype=torch.float64)
    if kind == "even":
        tokens = (u * rows).long()
    elif kind == "often":   # in proportion to 1 / rank
        tokens = (torch.exp(u * np.log(rows + 1.0)) - 1.0).long()
    elif kind == "one":
        tokens = torch.full(shape, rows // 2)
    else:                   # with tokens that are no row on either side
        tokens = (u * (rows + 4)).long() - 2
    return tokens.clamp(max=rows + 1).to(dtype).cuda()


# counts around 32 places and around two tiles of the sort (1024 each), with scanned counts beyond 32 of them; rows of one,
# two and three passes; widths of every number of lanes, beyond a slice, odd.  Of few rows and tokens one launch takes care
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("count,rows,width,kind", [
    (1, 1, 1, "even"), (1, 5, 7, "one"), (31, 3, 64, "even"), (32, 1, 33, "one"), (33, 2, 128, "even"), (64, 64, 20, "one"),
    (65, 9, 100, "beyond"), (1000, 32, 128, "often"), (2047, 2048, 17, "often"), (2048, 2047, 40, "even"), (2049, 4095, 8, "beyond"),
    (5000, 50000, 257, "often"), (4100, 3, 1023, "often"), (3000, 5, 2049, "one"), (900, 70, 5000, "often"), (70001, 300, 16, "often"),
    (66000, 100000, 24, "even"), (140000, 7, 12, "one"), (300, 5000000, 4, "even"), (70000, 5000000, 3, "often")])
def test_gradient(count, rows, width, kind, dtype):
    print(f"case: embedding gradient {count} tokens {rows} x {width} {kind} {dtype}", flush=True)
    check_gradient(make((count, width), dtype, 1), drawn((count,), rows, kind), rows, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,kind", [(9, "often"), (5000, "even"), (1, "one")])
def test_gradient_of_wide_rows(rows, kind, dtype):
    """So many lanes that float32 takes its longest tiles, bfloat16 the next."""
    print(f"case: embedding gradient of wide rows {rows} {kind} {dtype}", flush=True)
    check_gradient(make((17003, 1030), dtype, 1), drawn((17003,), rows, kind), rows, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["even", "often", "one", "beyond"])
def test_gradient_of_few_symbols(kind, dtype):
    """On both sides of what one launch takes, of 2 and 16 tokens a lane, and of a slice's columns."""
    for count, rows, width in ((1, 3, 5), (63, 512, 8), (64, 513, 8), (1023, 7, 31), (2047, 5, 33), (2049, 11, 64), (4096, 1, 65), (4097, 1, 40),
                               (5119, 5, 129), (5121, 5, 130), (16384, 16, 24), (16385, 17, 24), (9001, 100, 100)):
        print(f"case: embedding gradient of few {count} tokens {rows} x {width} {kind} {dtype}", flush=True)
        grad = make((count, 2 * width), dtype, 1)[:, :width]
        check_gradient(grad, drawn((count,), rows, kind, dtype=torch.int32), rows, -1.5)


@pytest.mark.parametrize("dtype,out", [(F32, BF16), (BF16, F32), (BF16, BF16)])
def test_gradient_types_and_strides(dtype, out):
    print(f"case: embedding gradient {dtype} to {out}", flush=True)
    grad = make((6, 50, 2, 40), dtype, 2)
    for view, lead in ((lambda t: t[:, :, 0], (6, 50)), (lambda t: t[:, ::2, 1].transpose(0, 1), (25, 6)), (lambda t: t[0, 0, 0].expand(7, 40), (7,)),
                       (lambda t: t[1:2, 3:4, 0], (1, 1)), (lambda t: t[:, 0, 0, :].t(), (40,))):
        check_gradient(view(grad), drawn(lead, 11, "often", 3, torch.int32), 11, -1.5, out)
    # tokens that are every second, gradients that start off 16 bytes
    flat = make(300 * 40 + 1, dtype, 3)
    check_gradient(flat[1:].view(300, 40), drawn((600,), 20, "beyond", 4)[::2], 20, 1.0, out)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 7), (40, 64), (9, 129), (30, 1000), (7, 2049), (3, 9000)])
def test_lookup(rows, width, dtype):
    print(f"case: embedding {rows} x {width} {dtype}", flush=True)
    table = make((rows, width), dtype)
    for shape, integer in (((), torch.int64), ((1,), torch.int32), ((3, 17), torch.int64), ((5, 0), torch.int32), ((1031,), torch.int64)):
        tokens = drawn(shape, rows, "beyond", 1, integer)
        for scale in (1.0, -3.7):
            out = ops.embedding(table, tokens, scale=scale)
            known = ((tokens >= 0) & (tokens < rows))[..., None]
            want = (table.float()[tokens.long().clamp(0, rows - 1)] * torch.tensor(scale, device="cuda") * known).to(dtype)
            assert out.dtype == dtype and out.shape == (*shape, width) and torch.equal(out, want)


def test_lookup_strides():
    print("case: embedding strides", flush=True)
    base = make((30, 3, 40), F32)
    tokens = drawn((60,), 30, "beyond", 2)
    for table in (base[:, 1], base[::2, 0], base[:, 0, ::2], base[0, 0].expand(30, 40), base[:, 2, 1:38]):
        rows = len(table)
        want = oo.embedding(numpy(table), tokens[::3].cpu().numpy())
        assert np.array_equal(numpy(ops.embedding(table, tokens[::3])), want), rows
    empty = ops.embedding(torch.empty(0, 8, device="cuda"), tokens)
    assert empty.shape == (60, 8) and (empty == 0).all()


def test_special_values_stay_in_their_rows():
    print("case: embedding special values", flush=True)
    grad, tokens = make((200, 24), F32), drawn((200,), 9, "often")
    at = int((tokens == 2).nonzero()[0])
    grad[at, 3], grad[at, 4] = float("nan"), float("inf")
    got = ops.embedding_backward(grad, tokens, 9)
    bad = ~torch.isfinite(got)
    assert torch.isnan(got[2, 3]) and torch.isinf(got[2, 4]) and bad.sum() == 2
    grad[tokens == 5] = float("nan")
    tokens[tokens == 5] = -7   # no row: its gradient is not looked at
    assert torch.equal(torch.isfinite(ops.embedding_backward(grad, tokens, 9)), ~bad)


def test_tokens_of_64_bits():
    """Tokens whose lower 32 bits would be a row."""
    print("case: embedding wide tokens", flush=True)
    tokens = torch.tensor([1, (1 << 32) + 1, -(1 << 32) + 1, -(1 << 63), 2], device="cuda")
    table = make((4, 8), F32)
    out = ops.embedding(table, tokens)
    assert torch.equal(out[0], table[1]) and torch.equal(out[4], table[2]) and (out[1:4] == 0).all()
    got = ops.embedding_backward(torch.ones(5, 8, device="cuda"), tokens, 4)
    assert got.sum(1).tolist() == [0.0, 8.0, 8.0, 0.0]


def test_gradient_offsets_beyond_32_bits():
    """A table and a batch of 2^31 + values each."""
    print("case: embedding offsets", flush=True)
    width, rows = 4096, (1 << 19) + 5
    tokens = torch.arange(rows, device="cuda").flip(0).to(torch.int32)
    row = make((1, width), BF16, 5)
    table = ops.embedding_backward(row.expand(rows, width), tokens, rows)
    assert torch.equal(table[-1], row[0]) and torch.equal(table[0], row[0]) and torch.equal(table[rows // 2], row[0])
    table[7], table[rows - 2] = 3.0, 5.0
    out = ops.embedding(table, tokens)
    assert (out[rows - 8] == 3.0).all() and (out[1] == 5.0).all() and torch.equal(out[0], row[0])


def test_symbols_empty_and_refused():
    print("case: embedding refusals", flush=True)
    table, tokens = make((5, 8), F32), torch.zeros(3, dtype=torch.int64, device="cuda")
    grad = make((3, 8), F32)
    none = ops.embedding_backward(grad[:0], tokens[:0], 5)
    assert none.shape == (5, 8) and (none == 0).all()
    assert ops.embedding_backward(grad, tokens, 0).shape == (0, 8)
    for call in (lambda: ops.embedding(table.half(), tokens), lambda: ops.embedding(table, tokens.float()), lambda: ops.embedding(table, tokens.cpu()),
                 lambda: ops.embedding(table[0], tokens), lambda: ops.embedding(table[:, :0], tokens), lambda: ops.embedding(table, [1, 2]),
                 lambda: ops.embedding(table.clone().requires_grad_(), tokens), lambda: ops.embedding(None, tokens),
                 lambda: ops.embedding_backward(grad, tokens[:2], 5), lambda: ops.embedding_backward(grad, tokens, -1),
                 lambda: ops.embedding_backward(grad, tokens, (1 << 31) - 1), lambda: ops.embedding_backward(grad, tokens, 5.0),
                 lambda: ops.embedding_backward(grad, tokens, 5, dtype=torch.float16), lambda: ops.embedding_backward(grad.half(), tokens, 5),
                 lambda: ops.embedding_backward(grad[:, :0], tokens, 5), lambda: ops.embedding_backward(grad, None, 5)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (33, 129), (2, 3, 1000), (70001,)])
def test_dropout(shape, dtype):
    print(f"case: dropout {shape} {dtype}", flush=True)
    x, residual = make(shape, dtype), make(shape, dtype, 1)
    for p, seed, stream, tick in ((0.1, 0, 0, 0), (0.5, (1 << 64) - 3, 5, 1 << 40), (0.0, 1, 2, 3), (1.0 - 2.0 ** -33, 4, 0, 9)):
        kept = torch.from_numpy(oo.dropout_kept(x.numel(), p, seed, stream, tick)).view(shape).cuda()
        factor = torch.tensor(1.0 / (1.0 - p), dtype=torch.float32, device="cuda")
        y = ops.dropout(x, p, seed, stream=stream, tick=tick)
        assert y.dtype == dtype and torch.equal(y, torch.where(kept, x.float() * factor, 0.0).to(dtype))
        held = torch.tensor([tick], device="cuda")
        assert torch.equal(y, ops.dropout(x, p, seed, stream=stream, tick=held))
        z = ops.dropout(x, p, seed, stream=stream, tick=tick, residual=residual)
        dropped = np.where(kept.cpu().numpy(), numpy(x) * float(factor), 0.0)
        want = numpy(residual) + dropped
        bound = 2 * ULP * (np.abs(dropped) + np.abs(want)) + ROUND[dtype] * np.abs(want)
        assert z.dtype == dtype and (np.abs(numpy(z) - want) <= bound).all()


def test_dropout_takes_places_not_strides():
    print("case: dropout strides", flush=True)
    base = make((40, 30, 3), F32)
    for x in (base.transpose(0, 1), base[::3], base[..., 1], base[0, 0].expand(40, 3), base.flatten()[1:]):
        assert torch.equal(ops.dropout(x, 0.3, 7), ops.dropout(x.contiguous(), 0.3, 7))
        residual = torch.ones_like(x).t() if x.dim() == 2 and x.shape[0] == x.shape[1] else torch.ones(1, device="cuda").expand(x.shape)
        assert torch.equal(ops.dropout(x, 0.3, 7, residual=residual), ops.dropout(x.contiguous(), 0.3, 7) + 1.0)


def test_dropout_of_special_values():
    """What is dropped is zero whatever it was."""
    print("case: dropout special values", flush=True)
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    kept = torch.from_numpy(oo.dropout_kept(4096, 0.5, 11)).cuda()
    y = ops.dropout(x, 0.5, 11)
    assert (y[~kept] == 0).all() and not torch.isfinite(y[kept]).any()


def test_dropout_beyond_32_bits():
    """The draws of places beyond 2^31 and of 2^32."""
    print("case: dropout offsets", flush=True)
    count = (1 << 32) + 64
    x = torch.ones(1, dtype=BF16, device="cuda").expand(count).contiguous()
    y = ops.dropout(x, 0.5, 3)
    for start in (1 << 31, (1 << 32) - 32, count - 32):
        want = [oo.counter_draw(3, 0, 0, i // 2) >> (32 * (i % 2)) & 0xFFFFFFFF for i in range(start, start + 32)]
        assert y[start:start + 32].tolist() == [2.0 if w >= 1 << 31 else 0.0 for w in want], start


def test_dropout_empty_and_refused():
    print("case: dropout refusals", flush=True)
    x = make((4, 8), F32)
    assert ops.dropout(x[:0], 0.5, 0).shape == (0, 8)
    for call in (lambda: ops.dropout(x.half(), 0.5, 0), lambda: ops.dropout(x, 1.0, 0), lambda: ops.dropout(x, -0.1, 0), lambda: ops.dropout(x, float("nan"), 0),
                 lambda: ops.dropout(x, 0.5, 1.5), lambda: ops.dropout(x, 0.5, 1 << 64), lambda: ops.dropout(x, 0.5, 0, stream="a"),
                 lambda: ops.dropout(x, 0.5, 0, tick=torch.zeros(2, dtype=torch.int64, device="cuda")), lambda: ops.dropout(x, 0.5, 0, tick=torch.zeros(1)),
                 lambda: ops.dropout(x, 0.5, 0, tick=torch.zeros(1, dtype=torch.int32, device="cuda")), lambda: ops.dropout(x, 0.5, 0, residual=x[:3]),
                 lambda: ops.dropout(x, 0.5, 0, residual=x.bfloat16()), lambda: ops.dropout(x.clone().requires_grad_(), 0.5, 0), lambda: ops.dropout(None, 0.5, 0)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("count", [1, 7, 4096, 8 * 256 * 4096 + 24581])
def test_dropout_in_place(count, dtype):
    """Through the C ABI, whose result may be its input or its residual: the same bits as in memory of its own."""
    print(f"case: dropout in place, {count} {dtype}", flush=True)
    x, residual = make((count,), dtype), make((count,), dtype, 1)
    for added in (None, residual):
        want = ops.dropout(x, 0.3, 5, stream=2, tick=9, residual=added)
        for name in ("x", "residual"):
            if name == "residual" and added is None:
                continue
            given = {"x": x.clone(), "residual": None if added is None else added.clone()}
            y = given[name]
            ops._call(0, ops.library().atlas_ops_dropout, given["x"].data_ptr(), None if added is None else given["residual"].data_ptr(), count,
                      ops.TYPES[dtype], 0.3, 5, 2, 9, None, y.data_ptr())
            assert torch.equal(y, want), name


# ------------------------------------------------------------- the gradient by sorting, whatever the tokens' number
# 601 rows are more than one launch takes, so few tokens are sorted too: counts around a tile of the sums (8 places, beyond
# 32 of them a list of its own) and of the sort (1024)
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("count", [1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 127, 129, 255, 257, 1023, 1024, 1025, 2049, 3000])
def test_gradient_by_sorting(count, dtype, out):
    print(f"case: sorted gradient of {count} tokens {dtype} to {out}", flush=True)
    for kind, width in (("one", 33), ("often", 20), ("even", 130), ("beyond", 7)):
        check_gradient(make((count, width), dtype, 1), drawn((count,), 601, kind), 601, -1.5, out)


@pytest.mark.parametrize("dtype,out", [(F32, BF16), (BF16, F32), (BF16, BF16)])
def test_gradient_by_sorting_of_strides(dtype, out):
    print(f"case: sorted gradient strides {dtype} to {out}", flush=True)
    grad = make((6, 50, 2, 40), dtype, 2)
    for view, lead in ((lambda t: t[:, :, 0], (6, 50)), (lambda t: t[:, ::2, 1].transpose(0, 1), (25, 6)), (lambda t: t[0, 0, 0].expand(7, 40), (7,)),
                       (lambda t: t[1:2, 3:4, 0], (1, 1)), (lambda t: t[:, 0, 0, :].t(), (40,))):
        check_gradient(view(grad), drawn(lead, 700, "often", 3, torch.int32), 700, -1.5, out)
    flat = make(300 * 40 + 1, dtype, 3)
    check_gradient(flat[1:].view(300, 40), drawn((600,), 700, "beyond", 4)[::2], 700, 1.0, out)


@pytest.mark.parametrize("dtype,count,rows,width", [(BF16, 32752, 50000, 1024), (F32, 9001, 50000, 512), (F32, 270001, 900, 8), (BF16, 520001, 900, 8)])
def test_gradient_by_sorting_in_each_length_of_tile(dtype, count, rows, width):
    """Tiles of 16 places with 128 lanes and with 16, of 8 with 128, of 32 with 16."""
    print(f"case: sorted gradient {count} tokens of {rows} x {width} {dtype}", flush=True)
    check_gradient(make((count, width), dtype, 1), drawn((count,), rows, "often"), rows, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_special_values_in_sorted_rows(dtype):
    """Non-finite values of rows within a tile, of rows that cross a few tiles and of one that crosses many."""
    print(f"case: sorted gradient special values {dtype}", flush=True)
    tokens = torch.cat([torch.full((n,), r) for r, n in ((2, 3), (5, 50), (9, 600), (300, 1), (600, 13))])
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(1))].cuda()
    grad = make((len(tokens), 24), dtype)
    clean = ops.embedding_backward(grad, tokens, 601)
    for row in (2, 5, 9, 300, 600):
        places = (tokens == row).nonzero().flatten().tolist()
        for at in (places[0], places[len(places) // 2], places[-1]):
            dirty = grad.clone()
            dirty[at, 3], dirty[at, 4] = float("nan"), -float("inf")
            got = ops.embedding_backward(dirty, tokens, 601)
            bad = ~torch.isfinite(got)
            assert torch.isnan(got[row, 3]) and got[row, 4] == -float("inf") and bad.sum() == 2 and torch.equal(got[~bad], clean[~bad])
    dirty = grad.clone()
    dirty[tokens == 9] = float("nan")
    gone = torch.where(tokens == 9, 601, tokens)   # no row any more: its gradients are not looked at
    got = ops.embedding_backward(dirty, gone, 601)
    assert (got[9] == 0).all() and torch.isfinite(got).all()


def test_sorted_tokens_of_64_bits():
    """Tokens whose lower 32 bits would be a row."""
    print("case: sorted wide tokens", flush=True)
    tokens = torch.tensor([1, (1 << 32) + 1, -(1 << 32) + 1, -(1 << 63), 2, 600, (1 << 33) + 600, 601, -1] * 40, device="cuda")
    got = ops.embedding_backward(torch.ones(len(tokens), 8, device="cuda"), tokens, 601)
    want = torch.zeros(601, device="cuda")
    want[[1, 2, 600]] = 40.0
    assert torch.equal(got, want[:, None].expand(601, 8))
