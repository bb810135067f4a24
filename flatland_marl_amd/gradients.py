"""Global norm of many gradient tensors, and clipping (flm_grad_clip): the norm of all elements together in one launch per
112 tensors, the scaling in as many.  The reference's optimizer never clips (src/agent.py:111-116); DQNAgent does when its
args hold max_grad_norm."""
from array import array
from operator import attrgetter

import torch

from ._lib import GRAD_MAX_TENSORS, GRAD_WORKSPACE, FlmError, launch

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _dense(t):
    """Whether the tensor's elements fill one stretch of memory, each place once, in whatever order."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


_place, _numel, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_device = torch.Tensor.get_device
_dtype, _layout, _shape = map(attrgetter, ("dtype", "layout", "shape"))


def _address(values):
    return values.buffer_info()[0]


def _inf_norm(norm_type):
    if float(norm_type) == 2.0:
        return 0
    if float(norm_type) == float("inf"):
        return 1
    raise ValueError("norm_type must be 2 or inf")


def _run(grads, max_norm, norm_type, outs):
    inf = _inf_norm(norm_type)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    count = len(grads)
    if count > GRAD_MAX_TENSORS:
        raise ValueError("%d gradient tensors, at most %d" % (count, GRAD_MAX_TENSORS))
    dev, index = grads[0].device, grads[0].get_device()
    if not grads[0].is_cuda:
        raise FlmError("gradients must live on a GPU: there is no CPU norm")
    if set(map(_device, grads)) != {index}:
        raise ValueError("gradients of several devices")
    if set(map(_layout, grads)) != {torch.strided}:
        raise ValueError("sparse gradients are not taken")
    types = list(map(_dtype, grads))
    if not set(types) <= DTYPES.keys():
        raise ValueError("gradients must be float32, bfloat16 or float16")
    straight = all(map(_contiguous, grads))
    if not straight and not all(map(_dense, grads)):
        raise ValueError("a gradient with gaps or repeated places between its elements")
    src, sizes = array("Q", map(_place, grads)), array("q", map(_numel, grads))
    kinds = array("i", map(DTYPES.__getitem__, types))
    dst = None
    if outs is not None:                                    # (whether any of them share memory is checked by the call)
        dst = src
        if outs is not grads:
            if list(map(_shape, outs)) != list(map(_shape, grads)) or list(map(_dtype, outs)) != types or \
                    set(map(_device, outs)) != {index}:
                raise ValueError("an output differs from its gradient in shape, type or device")
            if not (straight and all(map(_contiguous, outs))) and \
                    any(o.stride() != g.stride() for o, g in zip(outs, grads)):
                raise ValueError("an output differs from its gradient in strides")
            dst = array("Q", map(_place, outs))
    work = torch.empty(GRAD_WORKSPACE, dtype=torch.float64, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    launch(dev, "flm_grad_clip", _address(src), None if dst is None else _address(dst), _address(sizes), _address(kinds), count,
           float(max_norm), inf, work.data_ptr(), norm.data_ptr())
    return norm


def _listed(grads):
    return [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]


def grad_norm(grads, norm_type=2.0):
    """The norm of all elements of all tensors together: a float32 tensor [] on their device, nothing waited for.
    norm_type: 2 or inf (the largest absolute value).  None entries are skipped; no tensors: 0 (on the CPU)."""
    grads = _listed(grads)
    if not grads:
        _inf_norm(norm_type)
        return torch.zeros(())
    return _run(grads, 0.0, norm_type, None)


def clip_grad_norm_(grads, max_norm, norm_type=2.0, out=None):
    """Scales all tensors by min(1, max_norm / (norm + 1e-6)) in place and returns the norm they had, as grad_norm does.
    grads: gradient tensors (float32, bfloat16, float16, mixed at will; any size, no element twice), None entries are
    skipped.  out: a tensor for each gradient that receives the clipped values instead; the gradients stay as they are (an entry
    for every entry of grads, those of None entries are left alone, or one for every gradient).  A NaN norm makes every gradient
    NaN, an infinite one the finite ones zero (as the formula does: with an infinite max_norm as well it is NaN)."""
    outs = None
    if out is None or isinstance(grads, torch.Tensor):
        listed = _listed(grads)
        if out is not None:
            outs = _listed(out)
    else:
        if not isinstance(grads, (list, tuple)):
            grads = list(grads)
        if not isinstance(out, (list, tuple)):
            out = [out] if isinstance(out, torch.Tensor) else list(out)
        listed = _listed(grads)
        if len(out) == len(grads) != len(listed):           # one for one: what belongs to a None entry is left alone
            out = [o for g, o in zip(grads, out) if g is not None]
        outs = _listed(out)
        if listed and len(outs) != len(listed):
            raise ValueError("%d outputs for %d gradients" % (len(outs), len(listed)))
    if not listed:
        _inf_norm(norm_type)
        return torch.zeros(())
    return _run(listed, max_norm, norm_type, listed if outs is None else outs)
