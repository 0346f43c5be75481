"""Global norm of many gradient tensors and clipping by it, for the step between a backward pass
and the optimiser (the reference limits gradients there in its tracker network,
scripts/frontend/modules/clipping.py).

`global_norm` and `clip_by_global_norm` take the tensors, `clip_grad_norm_` parameters like
`torch.nn.utils.clip_grad_norm_`.  To clip a map's gradients inside the optimiser's step, without
writing them, pass `max_norm` to `surfel.SparseGaussianAdam.step`.

Everything stays on the device and on the current stream: nothing synchronises (except
`error_if_nonfinite`), so the calls can be captured into a graph.
"""
import ctypes

import torch

from . import _lib
from ._lib import VingsError, check, stream_ptr

_KINDS = {2.0: 0, float("inf"): 1}


def _dense(t):
    """Whether the elements of t fill one stretch of memory, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
        if size == 1:
            continue
        if stride != expected:
            return False
        expected *= size
    return True


def _checked(tensors, what):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise VingsError(f"{what}: no tensors given")
    dev = tensors[0].device
    for t in tensors:
        _lib.require_gpu_tensor(t, what)
        if t.layout != torch.strided:
            raise VingsError(f"{what}: sparse tensors are not supported")
        if t.dtype not in _lib.ELEM_TYPES:
            raise VingsError(f"{what}: float32, bfloat16 or float16 expected (got {t.dtype})")
        if t.device != dev:
            raise VingsError(f"{what}: all tensors must live on one device ({dev} and {t.device})")
        if not _dense(t):
            raise VingsError(f"{what}: a tensor with gaps or overlaps between its elements "
                             f"(shape {tuple(t.shape)}, strides {t.stride()}); pass a contiguous copy")
    return tensors, dev


def _kind(norm_type):
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise VingsError(f"norm_type must be 2 or inf (got {norm_type})")
    return kind


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _types(tensors):
    return (ctypes.c_int * len(tensors))(*[_lib.ELEM_TYPES[t.dtype] for t in tensors])


def norm_and_workspace(nbytes, dev):
    """(float32 scalar, address of `nbytes` of workspace) in one allocation: the workspace lives
    as long as the scalar, so of two captured graphs that share a memory pool neither is given
    the other's workspace while its norm is still to be read."""
    buf = torch.empty(2 + (nbytes + 3) // 4, dtype=torch.float32, device=dev)
    return buf[0], buf.data_ptr() + 8


def global_norm(tensors, norm_type=2.0):
    """Norm over all elements of `tensors` (a tensor or a sequence; float32, bfloat16 and float16
    may be mixed) as a float32 scalar on their device: the 2-norm, or the largest magnitude for
    norm_type=inf.  Sums are held in 64 bits: no overflow below the largest float32 norm.  A
    tensor given twice counts twice."""
    kind = _kind(norm_type)
    tensors, dev = _checked(tensors, "global_norm")
    L, n = _lib.lib(), len(tensors)
    numels = (ctypes.c_int64 * n)(*[t.numel() for t in tensors])
    with _lib.on_device(dev):
        nbytes = L.vings_grad_norm_workspace_bytes(n, numels)
        norm, ws = norm_and_workspace(nbytes, dev)
        check(L.vings_grad_norm(n, _pointers(tensors), numels, _types(tensors), kind, norm.data_ptr(),
                                ws, nbytes, stream_ptr(dev)), "vings_grad_norm")
    return norm


def clip_by_global_norm(tensors, max_norm, norm_type=2.0, out=None):
    """Scales `tensors` by min(1, max_norm / (norm + 1e-6)), norm = global_norm(tensors), and
    returns the norm.  In place, or into `out`: as many tensors of the same shapes and strides,
    each of its input's type or float32 (clipped float32 gradients of a bfloat16 backward pass),
    overlapping nothing else of the call.  In place a gradient that is short enough is left
    unwritten.  NaN gradients give a NaN norm and NaN results; an infinite norm gives zeros (and
    NaN where the gradient itself is infinite)."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise VingsError(f"max_norm must not be negative or NaN (got {max_norm})")
    tensors, dev = _checked(tensors, "clip_by_global_norm")
    if out is None:
        outs = tensors
    else:
        outs, out_dev = _checked(out, "clip_by_global_norm: out")
        if len(outs) != len(tensors) or out_dev != dev:
            raise VingsError("out must hold one tensor per gradient, on the gradients' device")
        for t, o in zip(tensors, outs):
            if t.shape != o.shape or (t.stride() != o.stride() and not (t.is_contiguous() and o.is_contiguous())):
                raise VingsError("out must have the shapes and strides of the gradients")
            if o.dtype not in (t.dtype, torch.float32):
                raise VingsError(f"a clipped {t.dtype} gradient is {t.dtype} or float32 (got {o.dtype})")
    L, n = _lib.lib(), len(tensors)
    numels = (ctypes.c_int64 * n)(*[t.numel() for t in tensors])
    ins, types = _pointers(tensors), _types(tensors)
    with _lib.on_device(dev):
        nbytes = L.vings_grad_norm_workspace_bytes(n, numels)
        norm, ws = norm_and_workspace(nbytes, dev)
        check(L.vings_grad_clip(n, ins, ins if out is None else _pointers(outs), numels, types,
                                types if out is None else _types(outs), kind, max_norm, norm.data_ptr(),
                                ws, nbytes, stream_ptr(dev)), "vings_grad_clip")
    torch.autograd.graph.increment_version(outs)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """`torch.nn.utils.clip_grad_norm_` for parameters on the GPU: clips their .grad in place by
    its global norm and returns the norm before clipping.  Parameters without a gradient are
    passed over (none at all: the norm is 0), a parameter given twice counts once.
    `error_if_nonfinite` reads the norm back and raises before anything is written."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    params = list({id(p): p for p in parameters}.values())
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=params[0].device if params else None)
    if error_if_nonfinite and not bool(torch.isfinite(global_norm(grads, norm_type))):
        raise VingsError("the gradients' norm is not finite")
    return clip_by_global_norm(grads, max_norm, norm_type)
