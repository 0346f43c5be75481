"""Rows of a table by integer id, scaled, with the gradient of the table: per-keyframe rows that
every splat reads through the keyframe that owns it (`SurfelMapper.globalkf_id`), or any other
table that a training loop indexes.

The gradient is summed by sorted ids in a fixed order: the same inputs give the same bits.  The
rows it touched come out as a mask, which is what `surfel.SparseGaussianAdam.step` takes as its
visibility: rows that no id named keep their values and moments.
"""
import torch

from . import _lib
from ._lib import VingsError, check, stream_ptr


_ID_TYPES = (torch.int32, torch.int64)


def _rows_2d(t):
    """t [..., D] as rows with unit column stride: (tensor, number of rows, row stride)."""
    D = t.shape[-1]
    n = t.numel() // D
    if t.is_contiguous():
        return t, n, D
    if t.dim() == 2 and (t.stride(1) == 1 or D == 1) and (n <= 1 or D <= t.stride(0) <= 1 << 20 or t.stride(0) == 0):
        return t, n, t.stride(0) if n > 1 else D
    t = t.contiguous()
    return t, n, D


def _check(t, ids, name):
    _lib.refuse_tangents((t,), name)
    if t.get_device() != ids.get_device() or t.get_device() < 0:
        _lib.require_gpu_tensor(t, name)
        _lib.require_gpu_tensor(ids, "ids")
        raise VingsError(f"{name} and ids must live on one device ({t.device} and {ids.device})")
    if t.dtype not in _lib.ELEM_TYPES:
        raise VingsError(f"{name}: float32, bfloat16 or float16 expected (got {t.dtype})")
    if ids.dtype not in _ID_TYPES:
        raise VingsError(f"ids must be int32 or int64 (got {ids.dtype})")
    if t.dim() < 1 or t.shape[-1] == 0:
        raise VingsError(f"{name} must have at least one column (got shape {tuple(t.shape)})")


def _check_touched(touched, num_rows, device):
    if touched is None:
        return
    if touched.dtype not in (torch.bool, torch.uint8) or touched.shape != (num_rows,) \
            or touched.device != device or not touched.is_contiguous():
        raise VingsError(f"touched must hold {num_rows} one-byte flags on {device}")


def _lookup(table, ids, scale):
    V, D = table.shape
    src, _, ld = _rows_2d(table)
    if ld == 0:
        src, ld = table.contiguous(), D
    flat = ids.contiguous()
    dev, dtype = table.device, table.dtype
    out = torch.empty((*ids.shape, D), dtype=dtype, device=dev)
    with _lib.on_device(dev):
        check(_lib.lib().vings_row_lookup(
            flat.numel(), V, D, src.data_ptr(), ld, _lib.ELEM_TYPES[dtype], flat.data_ptr(),
            flat.element_size(), scale, out.data_ptr(), stream_ptr(dev)), "vings_row_lookup")
    return out


def _lookup_backward(grad, ids, num_rows, scale, padding_id, out, touched, keep_touched):
    D = grad.shape[-1]
    src, n, ld = _rows_2d(grad)
    flat = ids.contiguous()
    if padding_id is None or not 0 <= padding_id < num_rows:
        padding_id = -1                  # names no row, like no padding id at all
    L, dev, et = _lib.lib(), grad.device, _lib.ELEM_TYPES[grad.dtype]
    with _lib.on_device(dev):
        nbytes = L.vings_row_lookup_backward_workspace_bytes(n, num_rows, D, et)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        check(L.vings_row_lookup_backward(
            n, num_rows, D, src.data_ptr(), ld, et, flat.data_ptr(), flat.element_size(),
            int(padding_id), scale, out.data_ptr(),
            _lib.ELEM_TYPES[out.dtype], None if touched is None else touched.data_ptr(),
            1 if keep_touched else 0, None if ws is None else ws.data_ptr(), nbytes, stream_ptr(dev)),
            "vings_row_lookup_backward")


class _LookupRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_id, touched):
        ctx.save_for_backward(ids)
        ctx.num_rows, ctx.scale, ctx.padding_id, ctx.touched = table.shape[0], scale, padding_id, touched
        return _lookup(table, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        _lib.refuse_tangents((g,), "the incoming gradient")
        rows = torch.empty((ctx.num_rows, g.shape[-1]), dtype=g.dtype, device=g.device)
        _lookup_backward(g, ids, ctx.num_rows, ctx.scale, ctx.padding_id, rows, ctx.touched, True)
        if ctx.touched is not None:
            torch.autograd.graph.increment_version(ctx.touched)
        return rows, None, None, None, None


def lookup_rows(table, ids, scale=1.0, padding_id=None, touched=None):
    """scale * table[ids] as a tensor of shape ids.shape + (D,) and table's type; differentiable
    in table (once, in reverse mode; forward-mode tangents are refused).

    table [V, D] float32 / bfloat16 / float16, its rows may lie in a wider array; ids int32 or
    int64 of any shape.  An id outside [0, V) names no row: zeros, and no gradient (-1 for a splat
    that no keyframe owns).  Ids equal to padding_id are looked up but give no gradient.  The
    product is taken in float32 and rounded once.

    touched: bool or uint8 [V].  The backward pass sets the entries of the rows that got a
    gradient and leaves the others as they are (several lookups of one step can mark one array;
    clear it once per step).

    Capturing a backward pass into a graph has PyTorch's own condition: no eager graph of the same
    leaves may be alive.  `lookup_rows_backward` has none."""
    _check(table, ids, "table")
    if table.dim() != 2:
        raise VingsError(f"table must be [rows, columns] (got shape {tuple(table.shape)})")
    _check_touched(touched, table.shape[0], table.device)
    if torch.is_grad_enabled() and table.requires_grad:
        return _LookupRows.apply(table, ids, float(scale), padding_id, touched)
    return _lookup(table, ids, float(scale))


def lookup_rows_backward(grad, ids, num_rows, scale=1.0, padding_id=None, out=None):
    """The gradient of `lookup_rows` without autograd: (rows [num_rows, D], touched [num_rows]
    bool), rows[v] = scale * sum of grad over the ids equal to v (zeros where there is none).

    grad: ids.shape + (D,); sums are float32 in a fixed order, rounded once to grad's type -- or
    to that of `out`, a contiguous [num_rows, D] tensor of grad's type or float32 that is
    overwritten and returned (float32 gradients for a float32 optimiser from bfloat16 ones)."""
    _check(grad, ids, "grad")
    num_rows = int(num_rows)
    if num_rows < 0:
        raise VingsError(f"num_rows must not be negative (got {num_rows})")
    if grad.shape[:-1] != ids.shape:
        raise VingsError(f"grad must have the shape of ids and one more dimension "
                         f"(got {tuple(grad.shape)} for ids {tuple(ids.shape)})")
    shape = (num_rows, grad.shape[-1])
    given = out is not None
    if not given:
        out = torch.empty(shape, dtype=grad.dtype, device=grad.device)
    elif tuple(out.shape) != shape or not out.is_contiguous() or out.device != grad.device \
            or out.dtype not in (grad.dtype, torch.float32):
        raise VingsError(f"out must be a contiguous {shape} tensor of {grad.dtype} or float32 on {grad.device}")
    touched = torch.empty(num_rows, dtype=torch.bool, device=grad.device)
    _lookup_backward(grad, ids, num_rows, float(scale), padding_id, out, touched, False)
    if given:
        torch.autograd.graph.increment_version(out)
    return out, touched
