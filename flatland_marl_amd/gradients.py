"""Global norm of many gradient tensors, and clipping (flm_grad_clip): the norm of all elements together in one launch per
112 tensors, the scaling in as many.  The reference's optimizer never clips (src/agent.py:111-116); DQNAgent does when its
args hold max_grad_norm."""
import ctypes as C
from operator import attrgetter

import torch

from ._lib import GRAD_MAX_TENSORS, GRAD_WORKSPACE, FlmError, call, ptr

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_dtype = attrgetter("dtype")


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


def _spans(tensors, sizes):
    return [(p, p + n * t.element_size()) for p, n, t in zip(map(torch.Tensor.data_ptr, tensors), sizes, tensors) if n]


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
    dev = grads[0].device
    if dev.type != "cuda":
        raise FlmError("gradients must live on a GPU: there is no CPU norm")
    if set(map(attrgetter("device"), grads)) != {dev}:
        raise ValueError("gradients of several devices")
    kinds = list(map(_dtype, grads))
    if not set(kinds) <= set(DTYPES):
        raise ValueError("gradients must be float32, bfloat16 or float16")
    if set(map(attrgetter("layout"), grads)) != {torch.strided}:
        raise ValueError("sparse gradients are not taken")
    if not all(map(_dense, grads)):
        raise ValueError("a gradient with gaps or repeated places between its elements")
    sizes = list(map(torch.Tensor.numel, grads))
    src = (C.c_void_p * count)(*map(torch.Tensor.data_ptr, grads))
    dst = None
    if outs is not None:
        spans = _spans(grads, sizes)
        dst = src
        if outs is not grads:
            if len(outs) != count:
                raise ValueError("as many outputs as gradients expected")
            for g, o in zip(grads, outs):
                if o.shape != g.shape or o.dtype != g.dtype or o.device != dev or \
                        (not (o.is_contiguous() and g.is_contiguous()) and o.stride() != g.stride()):
                    raise ValueError("an output differs from its gradient in shape, type, device or strides")
            dst = (C.c_void_p * count)(*map(torch.Tensor.data_ptr, outs))
            # (an output that is its own gradient's memory counts once)
            spans = spans + [s for s, g in zip(_spans(outs, sizes), spans) if s != g]
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("gradients (or their outputs) share memory: an element would be scaled twice")
    work = torch.empty(GRAD_WORKSPACE, dtype=torch.float64, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        call("flm_grad_clip", src, dst, (C.c_int64 * count)(*sizes), (C.c_int32 * count)(*[DTYPES[k] for k in kinds]), count,
             float(max_norm), inf, ptr(work), norm.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
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
    skipped.  out: a tensor for each gradient that receives the clipped values instead; the gradients stay as they are.
    A NaN norm makes every gradient NaN, an infinite one the finite ones zero."""
    outs = None
    listed = _listed(grads)
    if out is not None:
        outs = [out] if isinstance(out, torch.Tensor) else [o for o in out if o is not None]
    if not listed:
        _inf_norm(norm_type)
        return torch.zeros(())
    return _run(listed, max_norm, norm_type, listed if outs is None else outs)
