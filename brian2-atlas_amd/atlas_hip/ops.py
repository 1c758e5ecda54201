"""Operators of sequence layers on the MI355X: normalisation, layers of plastic synapses, the embedding of
symbols, dropout and the orthogonalised weight update.

Where ``rsnn`` trains one fixed recurrent network, these are the parts around a recurrent layer of
one's own: ``embedding`` for inputs that are symbols, ``layer_norm`` for its currents or ``rms_norm`` for a stream of
several layers, ``delta_rule`` and ``linear_attention`` as layers whose synapses decay and learn within a sequence
(``delta_rule_step`` and ``linear_attention_step`` for one tick of a stream), ``dropout``, and ``muon_update`` for its
dense matrices.  They take and return torch tensors on the GPU.  Each call enqueues hand-written kernels of
libatlas_ops_hip.so on the current stream of the tensors' device and returns without waiting;
workspaces come from torch's allocator.  Gradients are explicit calls, as the trainers' are: a tensor that
autograd follows is refused unless gradients are disabled, and so is a dual tensor of forward mode.  There is
no CPU fallback.

Invalid arguments raise ``ValueError``, a missing library ``NativeUnavailable``, a failed launch
``NativeError``.  Tensors may have any strides: what the kernels cannot address (a last axis that is
not contiguous) is copied first, except where a call updates a tensor in place, which has to be contiguous.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from pathlib import Path

import torch
from torch.autograd import forward_ad

from .native import NativeError, NativeUnavailable

LIBRARY = Path(__file__).resolve().parent.parent / "libatlas_ops_hip.so"
EXPORTS = ["atlas_ops_layer_norm", "atlas_ops_layer_norm_workspace", "atlas_ops_layer_norm_backward",
           "atlas_ops_orthogonalize_workspace", "atlas_ops_orthogonalize", "atlas_ops_delta_step",
           "atlas_ops_delta_workspace", "atlas_ops_delta_forward", "atlas_ops_delta_backward_workspace",
           "atlas_ops_delta_backward", "atlas_ops_rms_norm", "atlas_ops_rms_norm_workspace", "atlas_ops_rms_norm_backward",
           "atlas_ops_embedding", "atlas_ops_embedding_workspace", "atlas_ops_embedding_backward", "atlas_ops_dropout",
           "atlas_ops_linear_step", "atlas_ops_linear_workspace", "atlas_ops_linear_forward",
           "atlas_ops_linear_backward_workspace", "atlas_ops_linear_backward"]
TYPES = {torch.float32: 0, torch.bfloat16: 1}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_KEY = 128
INVALID = 7  # the entry points' code of an invalid argument

# the C structures of atlas_ops.h, packed as the ABI lays them out
_ROWS = struct.Struct("@P3q")
_ORTHOGONAL = struct.Struct("@P5q3P4i4f3f")
_DELTA = struct.Struct("@5P15q2P6q3if")
_lib = None
_local = threading.local()


def library() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIBRARY.exists():
            raise NativeUnavailable(f"{LIBRARY} is not built (run __graft_entry__.build())")
        lib = ctypes.CDLL(str(LIBRARY))
        vp, i64, i32, f32, text = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_char_p
        err = [vp, ctypes.c_size_t]
        lib.atlas_ops_layer_norm.argtypes = [text, i64, i64, i32, vp, vp, i32, f32, vp, vp, vp, vp, *err]
        lib.atlas_ops_layer_norm_workspace.argtypes = [i64, i64, i32]
        lib.atlas_ops_layer_norm_backward.argtypes = [text, text, i64, i64, i32, vp, i32, vp, vp, vp, vp, vp, vp, vp, *err]
        lib.atlas_ops_orthogonalize_workspace.argtypes = [i64, i64, i64]
        lib.atlas_ops_orthogonalize.argtypes = [text, vp, vp, *err]
        lib.atlas_ops_delta_step.argtypes = [text, vp, vp, vp, *err]
        lib.atlas_ops_delta_workspace.argtypes = [text, i32]
        lib.atlas_ops_delta_forward.argtypes = [text, i32, vp, vp, vp, vp, *err]
        lib.atlas_ops_delta_backward_workspace.argtypes = [text]
        lib.atlas_ops_delta_backward.argtypes = [text, vp, vp, text, vp, vp, vp, vp, vp, vp, vp, vp, vp, *err]
        f64, u64 = ctypes.c_double, ctypes.c_uint64
        lib.atlas_ops_rms_norm.argtypes = [text, text, i64, i64, i32, vp, i32, f32, vp, vp, vp, vp, vp, *err]
        lib.atlas_ops_rms_norm_workspace.argtypes = [i64, i64, i32]
        lib.atlas_ops_rms_norm_backward.argtypes = [text, text, text, i64, i64, i32, vp, i32, vp, vp, vp, vp, vp, *err]
        lib.atlas_ops_embedding.argtypes = [vp, i64, i64, i64, i32, vp, i32, i64, f32, vp, vp, *err]
        lib.atlas_ops_embedding_workspace.argtypes = [i64, i64, i64, i32]
        lib.atlas_ops_embedding_backward.argtypes = [text, vp, i32, i64, i64, i64, i32, i32, f32, vp, vp, vp, *err]
        lib.atlas_ops_dropout.argtypes = [vp, vp, i64, i32, f64, u64, u64, u64, vp, vp, vp, *err]
        lib.atlas_ops_linear_step.argtypes = [text, vp, vp, vp, *err]
        lib.atlas_ops_linear_workspace.argtypes = [text, i32]
        lib.atlas_ops_linear_forward.argtypes = [text, i32, vp, vp, vp, vp, *err]
        lib.atlas_ops_linear_backward_workspace.argtypes = [text]
        lib.atlas_ops_linear_backward.argtypes = [text, vp, vp, text, vp, vp, vp, vp, vp, i32, vp, vp, vp, *err]
        for name in EXPORTS:
            getattr(lib, name).restype = i64 if name.endswith("_workspace") else i32
        _lib = lib
    return _lib


def _call(device: int, entry, *args) -> None:
    """Runs one entry point on the device's current stream."""
    try:
        buffer, address = _local.error
    except AttributeError:
        buffer = ctypes.create_string_buffer(512)
        buffer, address = _local.error = (buffer, ctypes.addressof(buffer))
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch._C._cuda_getDevice() == device:
        rc = entry(*args, stream, address, 512)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream, address, 512)
    if rc:
        message = buffer.value.decode(errors="replace")
        raise ValueError(message) if rc == INVALID else NativeError(rc, message)


def _tensor(t, name: str, device=None, types=TYPES, shape=None):
    """The checks every tensor passes; returns its device's index."""
    index = t.get_device() if isinstance(t, torch.Tensor) else -1
    if index < 0:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if t.dtype not in types:
        raise ValueError(f"{name} is {t.dtype}, expected {' or '.join(str(x) for x in types)}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: gradients are explicit here, call under torch.no_grad()")
    if t.is_neg():
        raise ValueError(f"{name} is a view that negates what its memory holds: pass {name}.resolve_neg()")
    # forward mode: a level is open only within forward_ad.dual_level(), and disabled within an autograd.Function
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent: forward-mode derivatives are not computed here")
    if device is not None and index != device:
        raise ValueError(f"{name} is on GPU {index}, expected {device}")
    return index


_F32, _I32, _I64, _U8 = {torch.float32: 0}, {torch.int32: 0}, {torch.int64: 0}, {torch.uint8: 0}
_SAME = {t: {t: 0} for t in TYPES}


def _span(t):
    """From t's first element to its last, in elements."""
    return 1 + sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))


def _overlap(a, b):
    """Whether the memory from a's first element to its last and that of b have bytes in common."""
    start, other = a.data_ptr(), b.data_ptr()
    return start < other + _span(b) * b.element_size() and other < start + _span(a) * a.element_size()


def _empty(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _last(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _near(t):
    """(batch, time, ...) with tokens as near to one another as linear attention in chunks has them."""
    return t if t.stride(1) <= 1 << 24 or t.shape[1] == 1 else t.contiguous()


def _workspace(size: int, like):
    return torch.empty(size, dtype=torch.uint8, device=like.device)


# ------------------------------------------------------------------------------ layer normalisation
def _rows(x, rows, width):
    """x as rows of its last axis: the packed AtlasRows and the tensor it points into (a contiguous copy
    where the leading axes are not one or two strides)."""
    if x.is_contiguous():
        return _ROWS.pack(x.data_ptr(), rows, 0, width), x
    if width == 1 or x.stride(-1) == 1:
        axes = []  # (size, stride) from the innermost, neighbours joined
        for size, stride in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if size == 1:
                continue
            if axes and stride == axes[-1][0] * axes[-1][1]:
                axes[-1] = (axes[-1][0] * size, axes[-1][1])
            else:
                axes.append((size, stride))
        if len(axes) <= 2:
            axes += [(1, 0)] * (2 - len(axes))
            return _ROWS.pack(x.data_ptr(), axes[0][0], axes[1][1], axes[0][1]), x
    return _rows(x.contiguous(), rows, width)


_NORM_WEIGHTS = {torch.float32: {torch.float32: 0}, torch.bfloat16: TYPES}


def _norm_weights(x, width, weight, bias, device):
    """weight and bias, contiguous, and the code of their type."""
    types, code = _NORM_WEIGHTS[x.dtype], 0
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _tensor(t, name, device, types)
            if t.dim() != 1 or t.numel() != width:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(width,)}")
            code = types[t.dtype]
    if weight is not None:
        if bias is not None and weight.dtype != bias.dtype:
            raise ValueError("weight and bias must have the same type")
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return weight, bias, code


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, statistics: bool = False):
    """``(x - mean) * rstd * weight + bias`` over the last axis, ``rstd = 1 / sqrt(variance + eps)``.

    x: float32 or bfloat16; weight and bias: float32 or x's type.  Returns y, contiguous and of x's type; with
    ``statistics`` (y, mean, rstd), which ``layer_norm_backward`` takes, as float32 of x's leading shape."""
    device = _tensor(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError("x needs a last axis to normalise")
    weight, bias, code = _norm_weights(x, width, weight, bias, device)
    y = _empty(x)
    mean = rstd = None
    if statistics:
        mean, rstd = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=x.device).unbind()
    rows = x.numel() // width
    if rows:
        packed, keep = _rows(x, rows, width)
        _call(device, library().atlas_ops_layer_norm, packed, rows, width, TYPES[x.dtype],
              None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), code, eps,
              y.data_ptr(), mean.data_ptr() if statistics else None, rstd.data_ptr() if statistics else None)
    return (y, mean, rstd) if statistics else y


def layer_norm_backward(grad, x, weight, mean, rstd, *, sums: bool = True):
    """The gradients (dx, dweight, dbias) of ``layer_norm`` from that of its result.

    weight may be None (all ones; dweight and dbias are then float32).  Without ``sums`` dweight and dbias are
    None.  The sums over the rows are taken in float32 in a fixed order: the same bits on every run."""
    device = _tensor(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError("x needs a last axis to normalise")
    _tensor(grad, "grad", device, _SAME[x.dtype], x.shape)
    weight, _, code = _norm_weights(x, width, weight, None, device)
    wtype = torch.float32 if weight is None else weight.dtype
    lead = x.shape[:-1]
    _tensor(mean, "mean", device, _F32, lead)
    _tensor(rstd, "rstd", device, _F32, lead)
    rows, type_ = x.numel() // width, TYPES[x.dtype]
    dx = _empty(x)
    dweight = dbias = workspace = None
    lib = library()
    if sums:
        dweight, dbias = torch.empty((2, width), dtype=wtype, device=x.device).unbind()
        workspace = _workspace(lib.atlas_ops_layer_norm_workspace(rows, width, type_), x)
    if rows or sums:
        packed_grad, keep_grad = _rows(grad, rows, width) if rows else (None, None)
        packed, keep = _rows(x, rows, width) if rows else (None, None)
        mean, rstd = mean.contiguous(), rstd.contiguous()
        _call(device, lib.atlas_ops_layer_norm_backward, packed_grad, packed, rows, width, type_,
              None if weight is None else weight.data_ptr(), code, mean.data_ptr(), rstd.data_ptr(),
              dx.data_ptr(), dweight.data_ptr() if sums else None, dbias.data_ptr() if sums else None,
              workspace.data_ptr() if sums else None)
    return dx, dweight, dbias


# --------------------------------------------------------- root-mean-square norm of a stream
def _rms_arguments(x, weight, residual):
    """The device, width and rows of x and the checked weight with its type's code."""
    device = _tensor(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError("x needs a last axis to normalise")
    if residual is not None:
        _tensor(residual, "residual", device, _SAME[x.dtype], x.shape)
    weight, _, code = _norm_weights(x, width, weight, None, device)
    return device, width, x.numel() // width, weight, code


def _rms_forward(device, x, residual, rows, width, weight, code, eps, y, scale, total, rstd):
    packed, keep = _rows(x, rows, width)
    added, keep_added = (None, None) if residual is None else _rows(residual, rows, width)
    _call(device, library().atlas_ops_rms_norm, packed, added, rows, width, TYPES[x.dtype],
          None if weight is None else weight.data_ptr(), code, eps, y.data_ptr(), None if scale is None else scale.data_ptr(),
          None if total is None else total.data_ptr(), None if rstd is None else rstd.data_ptr())


def rms_norm(x, weight=None, residual=None, *, eps: float = 1e-5, statistics: bool = False):
    """``total * rstd * weight`` over the last axis, ``total = x + residual`` (rounded to x's type; x alone without a
    residual), ``rstd = 1 / sqrt(mean(total ** 2) + eps)``.

    x: float32 or bfloat16; residual: of x's shape and type; weight: float32 or x's type.  Returns y, or (y, total) with a
    residual, both contiguous and of x's type; ``statistics`` adds rstd at the end, float32 of x's leading shape, which
    ``rms_norm_backward`` takes.  The squares are summed in float32: where that is infinite, rstd is 0."""
    device, width, rows, weight, code = _rms_arguments(x, weight, residual)
    y = _empty(x)
    total = None if residual is None else _empty(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if statistics else None
    if rows:
        _rms_forward(device, x, residual, rows, width, weight, code, eps, y, None, total, rstd)
    if residual is None and not statistics:
        return y
    return (y, *(t for t in (total, rstd) if t is not None))


def rms_norm_8bit(x, weight=None, residual=None, *, eps: float = 1e-5):
    """``rms_norm`` for a product of 8 bits: (values, scale), or (values, scale, total) with a residual.

    values: float8_e4m3fn, the norm's result over its row's scale, computed in float32 and then rounded; scale: float32 of x's
    leading shape, the row's largest magnitude / 448, at least 2^-126.  A NaN has no part in the scale.  The scale is infinite
    where the row's largest magnitude or its sum of squares in float32 is: an infinity, or values above about 1e19."""
    device, width, rows, weight, code = _rms_arguments(x, weight, residual)
    values = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    total = None if residual is None else _empty(x)
    if rows:
        _rms_forward(device, x, residual, rows, width, weight, code, eps, values, scale, total, None)
    return (values, scale) if residual is None else (values, scale, total)


def rms_norm_backward(grad, total, weight, rstd, *, grad_total=None, sums: bool = True):
    """The gradients (dx, dweight) of ``rms_norm`` from that of y; dx is that of x and of the residual alike.

    total: x + residual as returned (x without a residual); grad_total: the gradient of total from where the stream goes
    on, added to dx.  weight may be None (all ones; dweight is then float32).  Without ``sums`` dweight is None.  The sums
    over the rows are taken in float32 in a fixed order: the same bits on every run."""
    device = _tensor(total, "total")
    width = total.shape[-1] if total.dim() else 0
    if width < 1:
        raise ValueError("total needs a last axis to normalise")
    same = _SAME[total.dtype]
    _tensor(grad, "grad", device, same, total.shape)
    if grad_total is not None:
        _tensor(grad_total, "grad_total", device, same, total.shape)
    weight, _, code = _norm_weights(total, width, weight, None, device)
    _tensor(rstd, "rstd", device, _F32, total.shape[:-1])
    rows, type_ = total.numel() // width, TYPES[total.dtype]
    dx = _empty(total)
    dweight = workspace = None
    lib = library()
    if sums:
        dweight = torch.empty(width, dtype=torch.float32 if weight is None else weight.dtype, device=total.device)
        workspace = _workspace(lib.atlas_ops_rms_norm_workspace(rows, width, type_), total)
    if rows or sums:
        packed_grad, keep_grad = _rows(grad, rows, width) if rows else (None, None)
        packed, keep = _rows(total, rows, width) if rows else (None, None)
        packed_stream, keep_stream = _rows(grad_total, rows, width) if rows and grad_total is not None else (None, None)
        rstd = rstd.contiguous()
        _call(device, lib.atlas_ops_rms_norm_backward, packed_grad, packed, packed_stream, rows, width, type_,
              None if weight is None else weight.data_ptr(), code, rstd.data_ptr(), dx.data_ptr(),
              dweight.data_ptr() if sums else None, workspace.data_ptr() if sums else None)
    return dx, dweight


# ------------------------------------------------------------------------- symbols
_INTEGERS = {torch.int64: 1, torch.int32: 0}
MAX_TOKENS, MAX_ROW = 1 << 27, 1 << 20


def embedding(table, tokens, *, scale: float = 1.0):
    """``scale * table[tokens]``: (*tokens' shape, width), contiguous and of the table's type.

    table: (rows, width), float32 or bfloat16; tokens: int32 or int64 of any shape.  A token that is no row, as -1 in the
    padding of a batch, gives zeros."""
    device = _tensor(table, "table")
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError("table must be (rows, width)")
    _tensor(tokens, "tokens", device, _INTEGERS)
    rows, width = table.shape
    shape = (*tokens.shape, width)
    if not rows:
        return torch.zeros(shape, dtype=table.dtype, device=table.device)
    out = torch.empty(shape, dtype=table.dtype, device=table.device)
    if tokens.numel():
        table, tokens = _last(table), tokens.contiguous()
        _call(device, library().atlas_ops_embedding, table.data_ptr(), rows, width, table.stride(0), TYPES[table.dtype],
              tokens.data_ptr(), _INTEGERS[tokens.dtype], tokens.numel(), scale, out.data_ptr())
    return out


def embedding_backward(grad, tokens, rows: int, *, scale: float = 1.0, dtype=None):
    """The gradient of ``embedding``'s table of ``rows`` rows from that of its result: (rows, width), of ``dtype`` (float32 or
    bfloat16, by default grad's).

    Row r is the sum of the gradients of its tokens, in their order and in float32, zeros without any; tokens that are no
    row have no part.  The same bits on every run.  At most 2^27 tokens, rows below 2^31 - 1, width up to 2^20."""
    device = _tensor(grad, "grad")
    if not grad.dim() or grad.shape[-1] < 1:
        raise ValueError("grad needs a last axis, that of the table")
    _tensor(tokens, "tokens", device, _INTEGERS, grad.shape[:-1])
    width, count = grad.shape[-1], tokens.numel()
    dtype = grad.dtype if dtype is None else dtype
    if dtype not in TYPES:
        raise ValueError(f"dtype is {dtype}, expected {' or '.join(str(x) for x in TYPES)}")
    if not isinstance(rows, int) or not 0 <= rows < (1 << 31) - 1 or count > MAX_TOKENS or width > MAX_ROW:
        raise ValueError(f"a table of {rows} rows of {width} from {count} tokens: at most 2^27 tokens, rows below 2^31 - 1, width up to 2^20")
    table = torch.empty((rows, width), dtype=dtype, device=grad.device)
    if rows:
        lib = library()
        packed, keep = _rows(grad, count, width) if count else (None, None)
        tokens = tokens.contiguous()
        workspace = _workspace(lib.atlas_ops_embedding_workspace(count, rows, width, TYPES[grad.dtype]), grad)
        _call(device, lib.atlas_ops_embedding_backward, packed, tokens.data_ptr(), _INTEGERS[tokens.dtype], count, rows, width,
              TYPES[grad.dtype], TYPES[dtype], scale, table.data_ptr(), workspace.data_ptr())
    return table


def dropout(x, probability: float, seed: int, *, stream: int = 0, tick=0, residual=None):
    """``residual + (x / (1 - probability) where it is kept, else 0)``, contiguous and of x's type; the same call on the
    gradient of the result, without the residual, is the gradient of x.

    The mask is not stored: it follows from the place of a value in x and from seed, stream (a layer's number) and tick (a
    step's), whole numbers of 64 bits, by the simulator's counter generator (``splitmix64-counter-v1``), each draw of
    which serves two neighbouring values, 32 bits each.  tick may be an int64 tensor of one value on the GPU, which is read
    when the kernel runs: a captured graph draws anew where the tensor has been counted up.  probability: 0 or
    more, below 1, resolved to 2^-32."""
    device = _tensor(x, "x")
    if not 0.0 <= probability < 1.0:
        raise ValueError("probability must be 0 or more and below 1")
    if residual is not None:
        _tensor(residual, "residual", device, _SAME[x.dtype], x.shape)
        residual = residual.contiguous()
    at = None
    if isinstance(tick, torch.Tensor):
        _tensor(tick, "tick", device, _I64)
        if tick.numel() != 1:
            raise ValueError("tick must be one value")
        at, tick = tick, 0
    for name, n in (("seed", seed), ("stream", stream), ("tick", tick)):
        if not isinstance(n, int) or not -(1 << 63) <= n < 1 << 64:
            raise ValueError(f"{name} must be a whole number of 64 bits")
    y = _empty(x)
    if x.numel():
        x = x.contiguous()
        _call(device, library().atlas_ops_dropout, x.data_ptr(), None if residual is None else residual.data_ptr(), x.numel(),
              TYPES[x.dtype], probability, seed, stream, tick, None if at is None else at.data_ptr(), y.data_ptr())
    return y


# --------------------------------------------------------------------- the orthogonalised update
def _matrix(t, name):
    if t.dim() not in (2, 3):
        raise ValueError(f"{name} must be a matrix or a batch of matrices")
    batch = t.shape[0] if t.dim() == 3 else 1
    return batch, t.shape[-2], t.shape[-1]


def _orthogonalize(device, source, shape, *, momentum, factor, nesterov, steps, coefficients, eps, weight=None,
                   keep=0.0, rate=0.0):
    """Into weight, or a new tensor, which it returns."""
    if not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError("steps must be 1 to 64")
    if len(coefficients) != 3:
        raise ValueError("the iteration has three coefficients")
    batch, rows, columns = shape
    lib = library()
    size = lib.atlas_ops_orthogonalize_workspace(batch, rows, columns)
    if not size:
        raise ValueError(f"{batch} matrices of {rows} x {columns}: at most 65535, of 2^20 rows and columns, one side at most 16384")
    out = _empty(source) if weight is None else None
    if source.stride(-1) != 1:
        source = source.contiguous()
    workspace = _workspace(size, source)
    packed = _ORTHOGONAL.pack(source.data_ptr(), batch, rows, columns, source.stride(0) if source.dim() == 3 else 0,
                              source.stride(-2), 0 if momentum is None else momentum.data_ptr(),
                              0 if out is None else out.data_ptr(), 0 if weight is None else weight.data_ptr(),
                              TYPES[source.dtype], TYPES[source.dtype], int(nesterov), steps,
                              factor, eps, keep, rate, *coefficients)
    _call(device, lib.atlas_ops_orthogonalize, packed, workspace.data_ptr())
    return out


def orthogonalize(matrix, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """Moves the singular values of a matrix (or of each matrix of a batch) towards one.

    ``X = matrix / (|matrix|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with
    ``A = X X^T`` and ``coefficients`` (a, b, c).  The default coefficients raise small singular values fast and
    leave the large ones between about 0.7 and 1.2.  Computed to float32's accuracy for either type; the result
    is contiguous and of the matrix's type.  Coefficients that could raise a matrix of the iteration beyond 4000 are
    refused.  At most 65535 matrices, of 2^20 rows and columns, one side at most 16384."""
    device = _tensor(matrix, "matrix")
    shape = _matrix(matrix, "matrix")
    if not matrix.numel():
        return _empty(matrix)
    return _orthogonalize(device, matrix, shape, momentum=None, factor=0.0, nesterov=False, steps=steps,
                          coefficients=coefficients, eps=eps)


def muon_update(weight, gradient, momentum, *, learning_rate: float, factor: float = 0.95, weight_decay: float = 0.0,
                nesterov: bool = True, scale: float | None = None, steps: int = 5, coefficients=COEFFICIENTS,
                eps: float = 1e-7) -> None:
    """One step of the Muon optimiser on a dense matrix (or a batch of them), in place:

    ``momentum <- factor momentum + gradient``,
    ``weight <- (1 - learning_rate weight_decay) weight - learning_rate scale orthogonalize(u)``,
    u = ``gradient + factor momentum`` with ``nesterov``, else the momentum.  Weights are (source, target), as the
    trainers'; ``scale`` is by default ``sqrt(max(1, targets / sources))``.  weight and momentum: float32, contiguous;
    gradient: float32 or bfloat16.  The three must not share memory."""
    device = _tensor(weight, "weight", types=_F32)
    shape = _matrix(weight, "weight")
    _tensor(momentum, "momentum", device, _F32, weight.shape)
    _tensor(gradient, "gradient", device, TYPES, weight.shape)
    for name, t in (("weight", weight), ("momentum", momentum)):
        if not t.is_contiguous():
            raise ValueError(f"{name} is updated in place and must be contiguous")
    if not weight.numel():
        return
    if _overlap(weight, momentum):
        raise ValueError("weight, momentum and gradient must not share memory")
    if _overlap(gradient, weight) or _overlap(gradient, momentum):
        if _span(gradient) == gradient.numel():
            raise ValueError("weight, momentum and gradient must not share memory")
        gradient = gradient.contiguous()  # the others may lie in the gaps between its rows
    if scale is None:
        scale = math.sqrt(max(1.0, shape[2] / shape[1]))
    _orthogonalize(device, gradient, shape, momentum=momentum, factor=factor, nesterov=nesterov, steps=steps,
                   coefficients=coefficients, eps=eps, weight=weight, keep=1.0 - learning_rate * weight_decay,
                   rate=learning_rate * scale)
    torch.autograd.graph.increment_version((weight, momentum))


# --------------------------------------------------------------------------- the gated delta rule
class _Problem:
    """The checked arguments of a delta rule, or of linear attention: sizes, the packed AtlasDelta and the tensors behind it."""

    __slots__ = ("device", "batch", "time", "heads", "value_heads", "key", "value", "type", "scale", "packed", "tensors")

    def __init__(self, q, k, v, log_decay, beta, state, lengths, scale, time_axis: bool, linear: bool = False):
        device = _tensor(q, "q")
        same = _SAME[q.dtype]
        _tensor(v, "v", device, same)
        shape, out = q.shape, v.shape
        if len(shape) != 3 + time_axis or len(out) != len(shape):
            raise ValueError(f"q, k and v must be {'(batch, time, heads, width)' if time_axis else '(batch, heads, width)'}")
        _tensor(k, "k", device, same, shape)
        *lead, heads, key = shape
        *given, value_heads, value = out
        if given != lead:
            raise ValueError(f"v has leading shape {tuple(given)}, q {tuple(lead)}")
        if heads < 1 or value_heads < 1 or value_heads % heads:
            raise ValueError("the heads of v must be a multiple of those of q and k")
        if not 1 <= key <= MAX_KEY or value < 1:
            raise ValueError(f"the width of q and k must be 1 to {MAX_KEY}, that of v positive")
        if linear and value > MAX_KEY:
            raise ValueError(f"the width of v must be 1 to {MAX_KEY}")
        gates = out[:-1]
        shared = linear and isinstance(log_decay, torch.Tensor) and log_decay.dim() == 1
        if log_decay is not None:
            _tensor(log_decay, "log_decay", device, TYPES, (value_heads,) if shared else gates)
        if not linear:
            _tensor(beta, "beta", device, TYPES, gates)
        batch, time = lead[0], lead[1] if time_axis else 1
        if state is not None:
            _tensor(state, "state", device, _F32, (batch, value_heads, key, value))
        if lengths is not None:
            _tensor(lengths, "lengths", device, _I32, (batch,))
            lengths = lengths.contiguous()
        q, k, v = _last(q), _last(k), _last(v)
        if linear and time_axis:
            q, k, v = _near(q), _near(k), _near(v)

        def strides(t):  # a single token, whose stride may be anything, is nowhere near another
            s = t.stride()
            return s[:3] if time > 1 else (s[0], 0, s[2]) if time_axis else (s[0], 0, s[1])

        self.device, self.batch, self.time, self.heads, self.value_heads = device, batch, time, heads, value_heads
        self.key, self.value, self.type, self.scale = key, value, q.dtype, scale
        self.tensors = (q, k, v, log_decay, beta, state, lengths)
        self.packed = _DELTA.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if log_decay is None else log_decay.data_ptr(),
            0 if linear else beta.data_ptr(), *strides(q), *strides(k), *strides(v),
            *((0, 0, 0) if log_decay is None else (0, 0, log_decay.stride(0)) if shared else strides(log_decay)),
            *((0, 0, 0) if linear else strides(beta)), 0 if state is None else state.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
            batch, time, heads, value_heads, key, value, TYPES[q.dtype],
            0 if log_decay is None else TYPES[log_decay.dtype], 0 if linear else TYPES[beta.dtype],
            1.0 / math.sqrt(key) if scale is None else scale)


def delta_rule_step(q, k, v, log_decay, beta, state, *, scale: float | None = None):
    """One tick of the gated delta rule for every stream of a batch; ``state`` is updated in place.

    As ``delta_rule`` without the time axis: q, k (batch, heads, key), v (batch, value heads, value), log_decay
    and beta (batch, value heads), state float32 (batch, value heads, key, value), contiguous, of memory that the other
    tensors have no part in.  Returns out."""
    if state is None:
        raise ValueError("a step needs a state to update")
    p = _Problem(q, k, v, log_decay, beta, state, None, scale, False)
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    out = _empty(v)
    if p.batch:
        _call(p.device, library().atlas_ops_delta_step, p.packed, out.data_ptr(), state.data_ptr())
        torch.autograd.graph.increment_version(state)
    return out


# Sequences up to this length without a tape run token by token in one launch: a token costs what the longest of
# them takes alike, while the chunks' two kernels cost the same from one token to 64.  Measured against chunks, with
# 16 heads of 128 x 128 in bfloat16: 16 sequences of 8 tokens 26 us to 48, of 16 tokens 46 to 48; one sequence
# of 8 heads 16 us to 19 and 27 to 20; 256 sequences of 4 heads of 64 x 64 43 us to 59 and 80 to 59.
SHORT = 12


class _Tape:
    __slots__ = ("problem", "memory", "stream")

    def __init__(self, problem, memory, stream):
        self.problem, self.memory, self.stream = problem, memory, stream

    def split(self):
        """(tensors, rest): all that the tape holds on the GPU, some None, as autograd's saved tensors take it, and what ``join``
        needs besides.  Hold no other reference to the tape to let its memory go with theirs."""
        return (*self.problem.tensors, self.memory), (self.stream, self.problem.scale)

    @classmethod
    def join(cls, tensors, rest):
        """The tape of ``split``, whose tensors may have moved in the meantime, or been laid out anew."""
        if len(tensors) != 8:
            raise ValueError("tensors must be those of a tape's split()")
        *inputs, state, lengths, memory = tensors
        stream, scale = rest
        if isinstance(state, torch.Tensor):
            state = state.contiguous()
        problem = _Problem(*inputs, state, lengths, scale, True, cls is LinearTape)
        if problem.batch and problem.time:
            _tensor(memory, "the tape's memory", problem.device, _U8)
            lib = library()
            if memory.numel() != (lib.atlas_ops_linear_workspace if cls is LinearTape else lib.atlas_ops_delta_workspace)(problem.packed, True):
                raise ValueError("the tape's memory is not that of these tensors")
            memory = memory.contiguous() if memory.data_ptr() % 16 == 0 else memory.clone(memory_format=torch.contiguous_format)
        return cls(problem, memory, stream)


class DeltaTape(_Tape):
    """What ``delta_rule_backward`` needs of a forward pass: its inputs and the chunks' states.  The inputs
    must not change before the backward pass has run."""

    __slots__ = ()


def delta_rule(q, k, v, log_decay, beta, state=None, *, lengths=None, scale: float | None = None, tape: bool = False):
    """The gated delta rule over sequences: a layer whose synapses decay and learn while it runs.

    Every value head keeps a state S (key x value), at first ``state`` or zeros.  By token
    ``S <- exp(log_decay) S``, ``e = v - S^T k``, ``S <- S + beta k e^T``, ``out = scale S^T q``.

    q, k (batch, time, heads, key), v (batch, time, value heads, value): float32 or bfloat16, key up to 128; value
    head h uses the q and k of head ``h // (value heads / heads)``.  log_decay (None: no decay) and beta
    (batch, time, value heads): float32 or bfloat16; a log_decay of -inf empties the state.  state: float32 (batch,
    value heads, key, value).  lengths: int32 (batch,), tokens from a sequence's length on leave its state
    unchanged, whatever is in it, and give zeros.  scale: by default ``1 / sqrt(key)``.  A NaN or an infinity reaches its own
    and later tokens only.  At most 65535 sequences and value heads, values up to 2^20 wide.

    Returns (out, final state); with ``tape`` (out, final state, tape), the tape for ``delta_rule_backward``."""
    if state is not None and isinstance(state, torch.Tensor):
        state = state.contiguous()
    p = _Problem(q, k, v, log_decay, beta, state, lengths, scale, True)
    out = _empty(v)
    shape = (p.batch, p.value_heads, p.key, p.value)
    memory = None
    if not p.batch or not p.time:
        final = torch.zeros(shape, dtype=torch.float32, device=v.device) if state is None else state.clone()
    else:
        final = torch.empty(shape, dtype=torch.float32, device=v.device)
        lib = library()
        if p.time <= SHORT and not tape:
            _call(p.device, lib.atlas_ops_delta_step, p.packed, out.data_ptr(), final.data_ptr())
        else:
            memory = _workspace(lib.atlas_ops_delta_workspace(p.packed, tape), v)
            _call(p.device, lib.atlas_ops_delta_forward, p.packed, tape, out.data_ptr(), final.data_ptr(),
                  memory.data_ptr())
    if tape:
        return out, final, DeltaTape(p, memory, torch._C._cuda_getCurrentRawStream(p.device))
    return out, final


def delta_rule_backward(grad_out, grad_state, tape: DeltaTape) -> dict:
    """The gradients of ``delta_rule`` from those of out (of its type) and of the final state (float32, or None
    for zeros): a dict with ``q, k, v, log_decay, beta, state``, each of its input's type, None for an input that
    was not given.  Heads of q and k that value heads share get the sum.  The same bits on every run.  A NaN or an infinity
    of a used token may reach the gradients of every token of its sequence."""
    if not isinstance(tape, DeltaTape):
        raise ValueError("tape must be the one that delta_rule returned")
    p = tape.problem
    q, k, v, log_decay, beta, state, lengths = p.tensors
    _tensor(grad_out, "grad_out", p.device, _SAME[p.type], v.shape)
    if grad_state is not None:
        _tensor(grad_state, "grad_state", p.device, _F32, (p.batch, p.value_heads, p.key, p.value))
        grad_state = grad_state.contiguous()
    grad_out = _last(grad_out)

    def like(t):
        return None if t is None else _empty(t)

    grads = {"q": like(q), "k": like(k), "v": like(v), "log_decay": like(log_decay), "beta": like(beta),
             "state": like(state)}
    if not p.batch or not p.time:
        if state is not None:
            grads["state"] = torch.zeros_like(state) if grad_state is None else grad_state.clone()
        return grads
    if torch._C._cuda_getCurrentRawStream(p.device) != tape.stream:
        # this stream's kernels read the tape: its memory is not to be reused before they have
        stream = torch.cuda.current_stream(p.device)
        for t in (tape.memory, *p.tensors):
            if t is not None:
                t.record_stream(stream)
    lib = library()
    workspace = _workspace(lib.atlas_ops_delta_backward_workspace(p.packed), v)
    _call(p.device, lib.atlas_ops_delta_backward, p.packed, tape.memory.data_ptr(), grad_out.data_ptr(),
          struct.pack("@3q", *grad_out.stride()[:3]), None if grad_state is None else grad_state.data_ptr(),
          *(None if grads[n] is None else grads[n].data_ptr() for n in ("q", "k", "v", "log_decay", "beta", "state")),
          workspace.data_ptr())
    return grads


# --------------------------------------------------------------------------------- linear attention
def linear_attention_step(q, k, v, log_decay, state, *, scale: float | None = None):
    """One tick of linear attention for every stream of a batch; ``state`` is updated in place.

    As ``linear_attention`` without the time axis: q, k (batch, heads, key), v (batch, value heads, value), log_decay (batch,
    value heads) or (value heads,), state float32 (batch, value heads, key, value), contiguous, of memory that the other
    tensors have no part in.  Returns out."""
    if state is None:
        raise ValueError("a step needs a state to update")
    p = _Problem(q, k, v, log_decay, None, state, None, scale, False, True)
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    out = _empty(v)
    if p.batch:
        _call(p.device, library().atlas_ops_linear_step, p.packed, out.data_ptr(), state.data_ptr())
        torch.autograd.graph.increment_version(state)
    return out


# Sequences up to this length without a tape run token by token in one launch.  Token by token and in chunks: 4 tokens, 8 heads
# of 64, float32 6.7 and 8.4 us, 64 sequences of them 11.1 and 11.6, bfloat16 heads of 128 22 and 29; 8 tokens 10.4 and 8.6, 17
# and 12, 33 and 30.
SHORT_LINEAR = 5


class LinearTape(_Tape):
    """What ``linear_attention_backward`` needs of a forward pass: its inputs and the segments' states.  The inputs must
    not change before the backward pass has run."""

    __slots__ = ()


def linear_attention(q, k, v, log_decay=None, state=None, *, lengths=None, scale: float | None = None, tape: bool = False):
    """Linear attention with a decay by head: a layer whose synapses grow by Hebb's rule and decay while it runs.

    Every value head keeps a state S (key x value), at first ``state`` or zeros.  By token
    ``S <- exp(log_decay) S + k v^T``, ``out = scale S^T q``.

    q, k (batch, time, heads, key), v (batch, time, value heads, value): float32 or bfloat16, key and value up to 128; value
    head h uses the q and k of head ``h // (value heads / heads)``.  log_decay (None: no decay): float32 or bfloat16, (batch,
    time, value heads), or (value heads,) for a decay that every token of a head has; -inf empties the state.  state:
    float32 (batch, value heads, key, value).  lengths: int32 (batch,), tokens from a sequence's length on leave its
    state unchanged, whatever is in it, and give zeros.  scale: by default ``1 / sqrt(key)``.  A NaN or an infinity reaches
    its own and later tokens only.  At most 65535 sequences and value heads, 2^29 tokens.

    Returns (out, final state); with ``tape`` (out, final state, tape), the tape for ``linear_attention_backward``."""
    if state is not None and isinstance(state, torch.Tensor):
        state = state.contiguous()
    p = _Problem(q, k, v, log_decay, None, state, lengths, scale, True, True)
    out = _empty(v)
    shape = (p.batch, p.value_heads, p.key, p.value)
    memory = None
    if not p.batch or not p.time:
        final = torch.zeros(shape, dtype=torch.float32, device=v.device) if state is None else state.clone()
    else:
        final = torch.empty(shape, dtype=torch.float32, device=v.device)
        lib = library()
        if p.time <= SHORT_LINEAR and not tape:
            _call(p.device, lib.atlas_ops_linear_step, p.packed, out.data_ptr(), final.data_ptr())
        else:
            memory = _workspace(lib.atlas_ops_linear_workspace(p.packed, tape), v)
            _call(p.device, lib.atlas_ops_linear_forward, p.packed, tape, out.data_ptr(), final.data_ptr(), memory.data_ptr())
    if tape:
        return out, final, LinearTape(p, memory, torch._C._cuda_getCurrentRawStream(p.device))
    return out, final


def linear_attention_backward(grad_out, grad_state, tape: LinearTape) -> dict:
    """The gradients of ``linear_attention`` from those of out (of its type) and of the final state (float32, or None for
    zeros): a dict with ``q, k, v, log_decay, state``, each of its input's shape and type, None for an input that was
    not given.  Heads of q and k that value heads share get the sum, a decay by head that of its tokens.  The same
    bits on every run.  A NaN or an infinity of a used token may reach the gradients of every token of its sequence."""
    if not isinstance(tape, LinearTape):
        raise ValueError("tape must be the one that linear_attention returned")
    p = tape.problem
    q, k, v, log_decay, _, state, lengths = p.tensors
    _tensor(grad_out, "grad_out", p.device, _SAME[p.type], v.shape)
    if grad_state is not None:
        _tensor(grad_state, "grad_state", p.device, _F32, (p.batch, p.value_heads, p.key, p.value))
        grad_state = grad_state.contiguous()
    grad_out = _near(_last(grad_out))
    go = grad_out.stride()
    grads = {name: None if t is None else _empty(t)
             for name, t in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("state", state))}
    if not p.batch or not p.time:
        if log_decay is not None:
            grads["log_decay"].zero_()
        if state is not None:
            grads["state"] = torch.zeros_like(state) if grad_state is None else grad_state.clone()
        return grads
    if torch._C._cuda_getCurrentRawStream(p.device) != tape.stream:
        # this stream's kernels read the tape: its memory is not to be reused before they have
        stream = torch.cuda.current_stream(p.device)
        for t in (tape.memory, *p.tensors):
            if t is not None:
                t.record_stream(stream)
    lib = library()
    workspace = _workspace(lib.atlas_ops_linear_backward_workspace(p.packed), v)
    dq, dk, dv, decay, dstate = (None if g is None else g.data_ptr() for g in grads.values())
    _call(p.device, lib.atlas_ops_linear_backward, p.packed, tape.memory.data_ptr(), grad_out.data_ptr(),
          struct.pack("@3q", go[0], go[1] if p.time > 1 else 0, go[2]), None if grad_state is None else grad_state.data_ptr(), dq, dk, dv, decay,
          int(log_decay is not None and log_decay.dim() == 1), dstate, workspace.data_ptr())
    return grads
