"""Global norm of many gradient tensors and clipping by it, for the step between a backward pass
and the optimiser (the reference limits gradients there in its tracker network,
scripts/frontend/modules/clipping.py).

`global_norm` and `clip_by_global_norm` take the tensors, `clip_grad_norm_` parameters like
`torch.nn.utils.clip_grad_norm_`.  To clip a map's gradients inside the optimiser's step, without
writing them, pass `max_norm` to `surfel.SparseGaussianAdam.step`.

Everything stays on the device and on the current stream: nothing synchronises (except
`error_if_nonfinite`), so the calls can be captured into a graph.  The calls stand outside
autograd: a norm carries no gradient, and forward-mode tangents are refused.
"""
import array
import operator

import torch

from . import _lib
from ._lib import VingsError, check, stream_ptr

_KINDS = {2.0: 0, float("inf"): 1}


# (lists of hundreds of small tensors are bound by the host: a bound method mapped over the list
# costs a third of the same attribute in a loop)
_numel, _data_ptr = torch.Tensor.numel, torch.Tensor.data_ptr
_get_device, _is_contiguous = torch.Tensor.get_device, torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")


def _dense(t):
    """Whether the elements of t fill one stretch of memory, in whatever order of dimensions."""
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
        if size == 1:
            continue
        if stride != expected:
            return False
        expected *= size
    return True


class TensorList:
    """A checked list of tensors and the tables the C entry points take."""
    __slots__ = ("tensors", "device", "contiguous", "n", "numels", "pointers", "types")

    def __init__(self, tensors, what):
        self.tensors = tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        if not tensors:
            raise VingsError(f"{what}: no tensors given")
        _lib.refuse_tangents(tensors, what)
        self.device = tensors[0].device
        types = list(map(_dtype, tensors))
        kinds = set(types)
        if len(kinds) == 1:
            types = [_lib.ELEM_TYPES.get(types[0])] * len(types)
        else:
            types = list(map(_lib.ELEM_TYPES.get, types))
        if None in types or set(map(_get_device, tensors)) != {self.device.index}:
            self._refuse(what)
        try:
            self.contiguous = all(map(_is_contiguous, tensors))
            pointers = array.array("Q", map(_data_ptr, tensors))
        except RuntimeError:
            raise VingsError(f"{what}: sparse tensors are not supported") from None
        if not self.contiguous:
            for t in tensors:
                if not t.is_contiguous() and not _dense(t):
                    raise VingsError(f"{what}: a tensor with gaps or overlaps between its elements "
                                     f"(shape {tuple(t.shape)}, strides {t.stride()}); pass a contiguous copy")
        self.n = len(tensors)
        self.pointers, self.types = pointers, array.array("i", types)
        self.numels = array.array("q", map(_numel, tensors))

    def _refuse(self, what):
        for t in self.tensors:
            _lib.require_gpu_tensor(t, what)
            if t.dtype not in _lib.ELEM_TYPES:
                raise VingsError(f"{what}: float32, bfloat16 or float16 expected (got {t.dtype})")
            if t.device != self.device:
                raise VingsError(f"{what}: all tensors must live on one device ({self.device} and {t.device})")


def _address(table):
    return table.buffer_info()[0]


def _kind(norm_type):
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise VingsError(f"norm_type must be 2 or inf (got {norm_type})")
    return kind


def norm_and_workspace(nbytes, dev):
    """(float32 scalar, address of `nbytes` of workspace) in one allocation: the workspace lives
    as long as the scalar, so of two captured graphs that share a memory pool neither is given
    the other's workspace while its norm is still to be read."""
    buf = torch.empty(2 + (nbytes + 3) // 4, dtype=torch.float32, device=dev)
    return buf[0], buf.data_ptr() + 8


def global_norm(tensors, norm_type=2.0):
    """Norm over all elements of `tensors` (a tensor or a sequence; float32, bfloat16 and float16
    may be mixed) as a float32 scalar on their device: the 2-norm, or the largest magnitude for
    norm_type=inf.  It carries no gradient, whatever the tensors require.  Sums are held in 64
    bits: no overflow below the largest float32 norm.  A tensor given twice counts twice."""
    kind = _kind(norm_type)
    g = TensorList(tensors, "global_norm")
    L, numels = _lib.lib(), _address(g.numels)
    with _lib.on_device(g.device):
        nbytes = L.vings_grad_norm_workspace_bytes(g.n, numels)
        norm, ws = norm_and_workspace(nbytes, g.device)
        check(L.vings_grad_norm(g.n, _address(g.pointers), numels, _address(g.types), kind, norm.data_ptr(),
                                ws, nbytes, stream_ptr(g.device)), "vings_grad_norm")
    return norm


def clip_by_global_norm(tensors, max_norm, norm_type=2.0, out=None):
    """Scales `tensors` by min(1, max_norm / (norm + 1e-6)), norm = global_norm(tensors), and
    returns the norm.  In place, or into `out`: as many tensors of the same shapes and strides,
    each of its input's type or float32 (clipped float32 gradients of a bfloat16 backward pass),
    overlapping nothing else of the call.  Autograd does not see the scaling.  In place a gradient
    that is short enough is left unwritten.  NaN gradients give a NaN norm and NaN results; an
    infinite norm gives zeros (and NaN where the gradient itself is infinite), or NaN if max_norm is
    infinite too."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise VingsError(f"max_norm must not be negative or NaN (got {max_norm})")
    g = TensorList(tensors, "clip_by_global_norm")
    o = g
    if out is not None:
        o = TensorList(out, "clip_by_global_norm: out")
        if o.n != g.n or o.device != g.device:
            raise VingsError("out must hold one tensor per gradient, on the gradients' device")
        for t, u in zip(g.tensors, o.tensors):
            if t.shape != u.shape or (t.stride() != u.stride() and not (t.is_contiguous() and u.is_contiguous())):
                raise VingsError("out must have the shapes and strides of the gradients")
            if u.dtype not in (t.dtype, torch.float32):
                raise VingsError(f"a clipped {t.dtype} gradient is {t.dtype} or float32 (got {u.dtype})")
    L, numels = _lib.lib(), _address(g.numels)
    with _lib.on_device(g.device):
        nbytes = L.vings_grad_norm_workspace_bytes(g.n, numels)
        norm, ws = norm_and_workspace(nbytes, g.device)
        check(L.vings_grad_clip(g.n, _address(g.pointers), _address(o.pointers), numels, _address(g.types),
                                _address(o.types), kind, max_norm, norm.data_ptr(), ws, nbytes,
                                stream_ptr(g.device)), "vings_grad_clip")
    torch.autograd.graph.increment_version(o.tensors)
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
