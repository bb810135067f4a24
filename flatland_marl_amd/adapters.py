"""Low-rank adapters of many requests beside one shared projection (flm_group_rows, flm_adapter_linear,
flm_adapter_linear_backward).  The reference trains one network for all maps (src/main.py:95); with adapters the network
stays shared and every map (or whatever the caller tells apart) adds a correction of low rank to a dense layer."""
import torch

from ._lib import ADAPTER_MAX_RANK, GROUPS_MAX, FlmError, launch, size_of
from .gradients import DTYPES


class RowGroups:
    """Rows sorted by group: what group_rows returns and the adapter calls take.  One int32 buffer; n rows, n_groups."""

    def __init__(self, buf, n, n_groups):
        self.buf, self.n, self.n_groups = buf, n, n_groups

    @property
    def order(self):
        """[n] int32: row numbers, stably sorted by group, the rows without a group last."""
        return self.buf[:self.n]

    @property
    def keys(self):
        """[n] int32: the group of order[i], n_groups for none."""
        at = (self.n + 3) // 4 * 4
        return self.buf[at:at + self.n]

    @property
    def offsets(self):
        """[n_groups + 1] int32: the rows of group g are order[offsets[g]:offsets[g + 1]]."""
        at = (self.n + 3) // 4 * 8
        return self.buf[at:at + self.n_groups + 1]


def group_rows(ids, n_groups):
    """Sorts rows by their group on the device, nothing waited for.  ids [n] int32 or int64: 0..n_groups-1, any other value
    means the row has no group."""
    n_groups = int(n_groups)
    if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("ids [n] of int32 or int64 expected")
    if not 1 <= n_groups <= GROUPS_MAX:
        raise ValueError("n_groups must be 1..%d" % GROUPS_MAX)
    dev, n = ids.device, ids.numel()
    if dev.type != "cuda":
        raise FlmError("ids must live on a GPU: there is no CPU path")
    if n == 0:
        return RowGroups(torch.zeros(n_groups + 1, dtype=torch.int32, device=dev), 0, n_groups)
    if n > 1 << 30:
        raise ValueError("more than 2^30 rows")
    if not ids.is_contiguous():
        ids = ids.contiguous()
    buf = torch.empty(size_of("flm_group_rows_ints", n, n_groups), dtype=torch.int32, device=dev)
    need = size_of("flm_group_rows_workspace", n, n_groups)
    work = torch.empty(need, dtype=torch.int32, device=dev) if need else None
    launch(dev, "flm_group_rows", ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, n, n_groups, buf.data_ptr(),
           work.data_ptr() if need else None)
    return RowGroups(buf, n, n_groups)


def _rows(t, name, width, dev, kind):
    """Row stride of a 2-D operand whose rows are contiguous."""
    if t.dim() != 2 or t.shape[1] != width:
        raise ValueError("%s [., %d] expected" % (name, width))
    if t.dtype != kind or t.device != dev:
        raise ValueError("%s differs from x in type or device" % name)
    if t.stride(1) != 1 and width > 1:
        raise ValueError("the rows of %s must be contiguous" % name)
    return t.stride(0) if t.shape[0] > 1 else width


def _weights(x, weight, a, b, groups, scale):
    if x.dim() != 2 or x.dtype not in DTYPES:
        raise ValueError("x [n, K] of float32, bfloat16 or float16 expected")
    n, k = x.shape
    dev, kind = x.device, x.dtype
    if dev.type != "cuda":
        raise FlmError("x must live on a GPU: there is no CPU path")
    if a.dim() != 3 or b.dim() != 3 or a.shape[2] != k or b.shape[0] != a.shape[0] or b.shape[2] != a.shape[1] or \
            not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("contiguous a [E, r, K] and b [E, N, r] expected")
    if a.dtype != kind or b.dtype != kind or a.device != dev or b.device != dev:
        raise ValueError("a and b differ from x in type or device")
    e, r = a.shape[0], a.shape[1]
    if not 1 <= r <= ADAPTER_MAX_RANK:
        raise ValueError("rank must be 1..%d" % ADAPTER_MAX_RANK)
    if groups.n != n or groups.n_groups != e or groups.buf.device != dev:
        raise ValueError("groups of %d rows and %d adapters expected" % (n, e))
    if max(n, k, b.shape[1]) > 1 << 20 or min(k, b.shape[1]) < 1:
        raise ValueError("rows, inputs and outputs must be at most 2^20")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (e,) or scale.device != dev or not scale.is_contiguous():
            raise ValueError("scale: a number or float32 [E] on the device of x")
        scales = (scale.data_ptr(), 1.0)
    else:
        scales = (None, float(scale))
    return n, k, b.shape[1], r, e, scales, _rows(x, "x", k, dev, kind), \
        _rows(weight, "weight", k, dev, kind) if weight is not None else 0


def adapter_linear(x, weight, bias, a, b, groups, scale=1.0, keep_low=False):
    """y[i] = weight x[i] + bias + scale[e] * b[e] (a[e] x[i]) for the adapter e of row i (groups = group_rows(ids, E)); rows
    without an adapter get the projection alone.  x [n, K], weight [N, K], bias [N] or None, a [E, r, K], b [E, N, r], all
    of one type (float32, bfloat16, float16); scale: a number or float32 [E].  keep_low: returns (y, low) with low [n, r]
    float32 = a[e] x[i], which the backward pass takes.  Runs on the current stream; no autograd."""
    n, k, n_out, r, e, scales, ldx, ldw = _weights(x, weight, a, b, groups, scale)
    if weight.shape[0] != n_out:
        raise ValueError("weight [%d, %d] expected" % (n_out, k))
    if bias is not None and (bias.shape != (n_out,) or bias.dtype != x.dtype or bias.device != x.device or
                             not bias.is_contiguous()):
        raise ValueError("contiguous bias [%d] in the type and on the device of x expected" % n_out)
    dev = x.device
    y = torch.empty((n, n_out), dtype=x.dtype, device=dev)
    low = torch.empty((n, r), dtype=torch.float32, device=dev) if keep_low else None
    if n:
        work = torch.empty(size_of("flm_adapter_workspace", n, k, n_out, r, e, DTYPES[x.dtype]), dtype=torch.uint8, device=dev)
        launch(dev, "flm_adapter_linear", x.data_ptr(), ldx, weight.data_ptr(), ldw, bias.data_ptr() if bias is not None else None,
               a.data_ptr(), b.data_ptr(), groups.buf.data_ptr(), *scales, n, k, n_out, r, e, DTYPES[x.dtype], work.data_ptr(),
               y.data_ptr(), n_out, low.data_ptr() if keep_low else None)
    return (y, low) if keep_low else y


def adapter_linear_backward(dy, x, weight, a, b, groups, low, scale=1.0, need_dx=True, da=None, db=None):
    """Gradients (dx, da, db) of adapter_linear for the gradient dy [n, N] of y; the shared projection is held fixed.
    low: what adapter_linear kept.  need_dx = False: dx is None and weight is not read (None is taken).  da, db: contiguous
    tensors like a and b that receive the gradients (fresh ones by default); adapters without rows get zeros."""
    n, k, n_out, r, e, scales, ldx, ldw = _weights(x, weight if need_dx else None, a, b, groups, scale)
    if need_dx and weight.shape[0] != n_out:
        raise ValueError("weight [%d, %d] expected" % (n_out, k))
    dev = x.device
    lddy = _rows(dy, "dy", n_out, dev, x.dtype)
    if dy.shape[0] != n:
        raise ValueError("dy [%d, %d] expected" % (n, n_out))
    if low.shape != (n, r) or low.dtype != torch.float32 or low.device != dev or not low.is_contiguous():
        raise ValueError("low [%d, %d] float32 as adapter_linear keeps it expected" % (n, r))
    for name, t, like in (("da", da, a), ("db", db, b)):
        if t is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != dev or not t.is_contiguous()):
            raise ValueError("%s: a contiguous tensor like its parameter expected" % name)
    da = torch.empty_like(a) if da is None else da
    db = torch.empty_like(b) if db is None else db
    dx = torch.empty((n, k), dtype=x.dtype, device=dev) if need_dx else None
    if n == 0:
        da.zero_()
        db.zero_()
        return dx, da, db
    kind = DTYPES[x.dtype]
    work = torch.empty(size_of("flm_adapter_backward_workspace", n, k, n_out, r, e, kind, 1 if need_dx else 0), dtype=torch.uint8,
                       device=dev)
    launch(dev, "flm_adapter_linear_backward", dy.data_ptr(), lddy, x.data_ptr(), ldx, weight.data_ptr() if need_dx else None, ldw,
           a.data_ptr(), b.data_ptr(), groups.buf.data_ptr(), *scales, low.data_ptr(), n, k, n_out, r, e, kind, work.data_ptr(),
           dx.data_ptr() if need_dx else None, k, da.data_ptr(), db.data_ptr())
    return dx, da, db
