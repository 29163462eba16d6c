"""Latent rows as outputs: embedding lookup with scaling, and its gradient by
sorted ids (mfm_embedding_* in the C ABI).

The engine's scoring and training kernels gather latent rows by feature id and
add up their gradients per touched id without either leaving the device;
these calls hand both to a caller's own model on the same inputs: ids with one
value each, alone or as the rows of a canonical CSR
(``prep.prep_csr_device``), against a table of latent rows.

All calls take CUDA tensors on one device, run on ``stream`` (a
torch.cuda.Stream, default the current one of that device) and neither
synchronise nor copy to the host, so they can be captured into a CUDA graph.
Ids outside ``[0, n_rows)`` are padding: a zero row, no gradient. Every sum has a
fixed order: results are bitwise reproducible. The calls are not part of torch's
autograd: results carry no graph, whether or not an input requires a gradient, and
a backward pass is a call of its own (``embedding_grad``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class EmbeddingGrad(NamedTuple):
    """``table`` (n_rows, d); ``scale`` one value per entry, or None."""
    table: object
    scale: Optional[object]


class EmbeddingRows(NamedTuple):
    """The touched ids ``keys`` in ascending order and their gradient ``rows``, in
    min(n_entries, n_rows) places of which ``count`` (a 0-dim int64 tensor) are
    used: keys are -1 and rows 0 behind them. ``scale`` as in EmbeddingGrad."""
    keys: object
    rows: object
    count: object
    scale: Optional[object]


_STORAGE = {torch.float64: _lib.MFM_DTYPE_F64, torch.float32: _lib.MFM_DTYPE_F32,
            torch.bfloat16: _lib.MFM_DTYPE_BF16, torch.float16: _lib.MFM_DTYPE_F16}


def _fail(rc):
    if rc:
        raise (ValueError if rc < 0 else RuntimeError)(_lib.last_error())


def _one_device(first, *rest):
    """The device index that all tensors (None: not given) share."""
    if not first.is_cuda:
        raise ValueError("every tensor must be a CUDA tensor")
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise ValueError("every tensor must be a CUDA tensor on one device")
    return dev


def _matrix(name, t):
    """(pointer, rows, columns, row pitch) of a matrix with contiguous rows that do not overlap."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix with contiguous rows")
    n, d = t.shape
    pitch, step = t.stride()
    if d > 1 and step != 1:
        raise ValueError(f"{name} must be a matrix with contiguous rows")
    if n <= 1:
        pitch = max(d, 1)
    if pitch < d:
        raise ValueError(f"the rows of {name} must not overlap")
    return t.data_ptr(), n, d, pitch


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Nothing:
    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False


_NOTHING = _Nothing()


def _on(stream, dev):
    """(stream handle, context that allocates on it)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(dev), _NOTHING
    if stream.device.index != dev:
        raise ValueError("stream belongs to another device")
    return stream.cuda_stream, torch.cuda.stream(stream)


def _hold(stream, *tensors):
    """Keeps the memory of inputs of another stream until `stream` is done with them."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _entries(ids, scale, indptr, wide):
    kind = ids.dtype
    if not (kind is torch.int64 or kind is torch.int32) or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 or int64 tensor")
    if indptr is not None:
        if ids.dim() != 1:
            raise ValueError("ids must be 1-D with indptr")
        if (indptr.dtype != torch.int64 or indptr.dim() != 1 or not indptr.is_contiguous()
                or indptr.numel() < 1):
            raise ValueError("indptr must be a contiguous 1-D int64 tensor (n_out + 1)")
    if scale is not None:
        if scale.shape != ids.shape or not scale.is_contiguous():
            raise ValueError("scale must be contiguous and have the shape of ids")
        if scale.dtype != wide:
            raise ValueError(f"scale must be {wide}")
    return 1 if kind is torch.int64 else 0


def embedding_lookup(table, ids, scale=None, indptr=None, alpha: float = 1.0, out=None,
                     stream=None):
    """``alpha * scale[t] * table[ids[t]]`` for every id, or, with ``indptr`` (int64,
    n_out + 1), those rows summed over the entries of each CSR row.

    ``table`` (n_rows, d) is float64, float32, bfloat16 or float16 with
    contiguous rows of any pitch; ``ids`` int32 or int64 of any shape (1-D with
    ``indptr``); ``scale`` has their shape and is float64 for a float64 table, else
    float32. A float64 ``scale`` with a float32 table gives float64 arithmetic and a
    float64 result (the engine's default arithmetic). Returns ids.shape + (d,) or
    (n_out, d) in the table's type, sums rounded once; ``out`` (2-D for a 1-D
    ids) takes the result instead of a new tensor and must not overlap the
    inputs. A CSR row is summed by one group of lanes: rows of up to some thousand
    entries, or many of them, are what it is made for. Raises ValueError for invalid arguments, RuntimeError for CUDA
    failures.
    """
    code = _STORAGE.get(table.dtype)
    if code is None:
        raise ValueError("table must be float64, float32, bfloat16 or float16")
    wide = torch.float64 if table.dtype == torch.float64 else torch.float32
    kind = table.dtype
    if scale is not None and table.dtype == torch.float32 and scale.dtype == torch.float64:
        code, wide, kind = _lib.MFM_DTYPE_F32_F64, torch.float64, torch.float64
    ids64 = _entries(ids, scale, indptr, wide)
    tp, n_rows, d, ld = _matrix("table", table)
    if d < 1:
        raise ValueError("embedding width must be >= 1")
    dev = _one_device(table, ids, scale, indptr, out)
    n = ids.numel()
    n_out = n if indptr is None else indptr.numel() - 1
    s, ctx = _on(stream, dev)
    _hold(stream, table, ids, scale, indptr, out)
    if out is None:
        with ctx:
            out = table.new_empty((n_out, d), dtype=kind)
        op, ld_out = out.data_ptr(), d
        result = out if ids.dim() == 1 else out.view(ids.shape + (d,))
    else:
        if out.dtype != kind or tuple(out.shape) != (n_out, d):
            raise ValueError(f"out must be {kind} of shape {(n_out, d)}")
        result = out
        op, _, _, ld_out = _matrix("out", out)
    _fail(_lib.lib().mfm_embedding_lookup_device(
        code, dev, ids64, ids.data_ptr(), n, _ptr(indptr), n_out, _ptr(scale), float(alpha), tp,
        n_rows, d, ld, op, ld_out, s))
    return result


def _grad(grad, ids, n_rows, scale, indptr, alpha, table, dtype, stream, by_rows):
    code = _STORAGE.get(grad.dtype)
    if code is None:
        raise ValueError("grad must be float64, float32, bfloat16 or float16")
    halves = grad.dtype in (torch.bfloat16, torch.float16)
    wide = torch.float64 if grad.dtype == torch.float64 else torch.float32
    kind = grad.dtype if dtype is None else dtype
    if kind != grad.dtype and not (halves and kind == torch.float32):
        raise ValueError("dtype must be grad's, or float32 for bfloat16 and float16")
    ids64 = _entries(ids, scale, indptr, wide)
    n_rows = int(n_rows)
    if n_rows < 0:
        raise ValueError("n_rows must be >= 0")
    n = ids.numel()
    n_out = n if indptr is None else indptr.numel() - 1
    source = grad
    if grad.dim() > 2:  # a copy where the strides need one, made by the stream that reads it
        with _NOTHING if stream is None else torch.cuda.stream(stream):
            grad = grad.flatten(0, -2)
    elif grad.dim() == 1 and ids.dim() == 0:
        grad = grad[None]
    gp, given, d, ld = _matrix("grad", grad)
    if d < 1:
        raise ValueError("embedding width must be >= 1")
    if given != n_out:
        raise ValueError(f"grad must have one row per {'id' if indptr is None else 'CSR row'}")
    tp, ld_table = None, d
    if table is not None:
        if tuple(table.shape) != (n_rows, d):
            raise ValueError(f"table must have shape {(n_rows, d)}")
        if table.dtype == torch.float32 and grad.dtype == torch.float64:
            code = _lib.MFM_DTYPE_F32_F64
        elif table.dtype != grad.dtype:
            raise ValueError("table must have grad's type (or be float32 with a float64 grad)")
        tp, _, _, ld_table = _matrix("table", table)
    dev = _one_device(grad, ids, scale, indptr, table)
    L = _lib.lib()
    nbytes = L.mfm_embedding_grad_workspace_bytes(code, 1 if by_rows else 0, n, n_rows, d)
    s, ctx = _on(stream, dev)
    _hold(stream, source, grad, ids, scale, indptr, table)
    keys = rows = count = whole = d_scale = None
    with ctx:
        ws = grad.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        if by_rows:
            cap = min(n, n_rows)
            keys = ids.new_empty(cap)
            rows = grad.new_empty((cap, d), dtype=kind)
            count = grad.new_empty((), dtype=torch.int64)
        else:
            whole = grad.new_empty((n_rows, d), dtype=kind)
        if table is not None:
            d_scale = grad.new_empty(ids.shape, dtype=wide)
    # empty tensors have no address; the ABI tells its two results apart by theirs
    at = lambda t: None if t is None else (t.data_ptr() or 256)  # noqa: E731
    _fail(L.mfm_embedding_grad_device(
        code, _STORAGE[kind], dev, ids64, ids.data_ptr(), n, _ptr(indptr), n_out, _ptr(scale),
        float(alpha), gp, ld, tp, ld_table, n_rows, d, at(whole), at(keys), at(rows), at(count),
        _ptr(d_scale), _ptr(ws), nbytes, s))
    return whole, keys, rows, count, d_scale


def embedding_grad(grad, ids, n_rows: int, scale=None, indptr=None, alpha: float = 1.0, table=None,
                   dtype=None, stream=None) -> EmbeddingGrad:
    """Gradient of ``embedding_lookup`` over the whole table:
    ``d_table[i] = alpha * sum of scale[t] * grad[row(t)]`` over the entries with id i.

    ``grad`` has the lookup's result's shape; ``ids``, ``scale``, ``indptr`` and
    ``alpha`` are the lookup's (``scale`` float64 for a float64 grad, else float32).
    ``dtype`` torch.float32 keeps the sums of a bfloat16 or float16 grad in
    float32 instead of rounding them. With ``table`` (the lookup's) the gradient
    of ``scale`` is returned too: ``alpha * <grad[row(t)], table[ids[t]]>``.
    """
    whole, _, _, _, d_scale = _grad(grad, ids, n_rows, scale, indptr, alpha, table, dtype, stream,
                                    False)
    return EmbeddingGrad(whole, d_scale)


def embedding_grad_rows(grad, ids, n_rows: int, scale=None, indptr=None, alpha: float = 1.0,
                        table=None, dtype=None, stream=None) -> EmbeddingRows:
    """``embedding_grad`` of the touched rows only, as the engine's optimizers step
    them: their ids in ascending order and one gradient row each."""
    _, keys, rows, count, d_scale = _grad(grad, ids, n_rows, scale, indptr, alpha, table, dtype,
                                          stream, True)
    return EmbeddingRows(keys, rows, count, d_scale)
