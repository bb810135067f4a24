"""Low-rank adapters of many requests beside one shared projection (flm_group_rows, flm_adapter_linear,
flm_adapter_linear_backward).  The reference trains one network for all maps (src/main.py:95); with adapters the network
stays shared and every map (or whatever the caller tells apart) adds a correction of low rank to a dense layer."""
import torch

from ._lib import ADAPTER_MAX_RANK, GROUPS_MAX, FlmError, launch, size_of
from .gradients import DTYPES


SIZE_MAX = 1 << 20                                          # rows, inputs, outputs


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
    if not ids.is_cuda:
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
    shape = t.shape
    if len(shape) != 2 or shape[1] != width:
        raise ValueError("%s [., %d] expected" % (name, width))
    if t.dtype != kind or t.device != dev:
        raise ValueError("%s differs from x in type or device" % name)
    across, along = t.stride()
    if along != 1 and width > 1:
        raise ValueError("the rows of %s must be contiguous" % name)
    return across if shape[0] > 1 else width


def _weights(x, weight, a, b, groups, scale):
    kind, dev = x.dtype, x.device
    if x.dim() != 2 or kind not in DTYPES:
        raise ValueError("x [n, K] of float32, bfloat16 or float16 expected")
    n, k = x.shape
    if not x.is_cuda:
        raise FlmError("x must live on a GPU: there is no CPU path")
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("contiguous a [E, r, K] and b [E, N, r] expected")
    e, r, k_a = a.shape
    e_b, n_out, r_b = b.shape
    if k_a != k or e_b != e or r_b != r or not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("contiguous a [E, r, K] and b [E, N, r] expected")
    if a.dtype != kind or b.dtype != kind or a.device != dev or b.device != dev:
        raise ValueError("a and b differ from x in type or device")
    if not 1 <= r <= ADAPTER_MAX_RANK:
        raise ValueError("rank must be 1..%d" % ADAPTER_MAX_RANK)
    if groups.n != n or groups.n_groups != e or groups.buf.device != dev:
        raise ValueError("groups of %d rows and %d adapters expected" % (n, e))
    if not (n <= SIZE_MAX and 1 <= k <= SIZE_MAX and 1 <= n_out <= SIZE_MAX):
        raise ValueError("rows, inputs and outputs must be at most 2^20")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != (e,) or scale.device != dev or not scale.is_contiguous():
            raise ValueError("scale: a number or float32 [E] on the device of x")
        scales = (scale.data_ptr(), 1.0)
    else:
        scales = (None, float(scale))
    return n, k, n_out, r, e, scales, _rows(x, "x", k, dev, kind), \
        _rows(weight, "weight", k, dev, kind) if weight is not None else 0


def adapter_linear(x, weight, bias, a, b, groups, scale=1.0, keep_low=False, out=None):
    """y[i] = weight x[i] + bias + scale[e] * b[e] (a[e] x[i]) for the adapter e of row i (groups = group_rows(ids, E)); rows
    without an adapter get the projection alone.  x [n, K], weight [N, K], bias [N] or None, a [E, r, K], b [E, N, r], all
    of one type (float32, bfloat16, float16); scale: a number or float32 [E].  keep_low: returns (y, low) with low [n, r]
    float32 = a[e] x[i], which the backward pass takes.  out: a tensor [n, N] with contiguous rows that receives y (it may
    share no element with an input).  A result is finite where the formula's is; an infinite one may be NaN instead.  Runs on
    the current stream.  No autograd: where gradients are recorded, operands that require one are refused (torch.no_grad(), or
    detached operands, and adapter_linear_backward)."""
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        raise ValueError("adapter_linear records no graph: call it under torch.no_grad(), or with detached operands, and "
                         "adapter_linear_backward for the gradients")
    n, k, n_out, r, e, scales, ldx, ldw = _weights(x, weight, a, b, groups, scale)
    if weight.shape[0] != n_out:
        raise ValueError("weight [%d, %d] expected" % (n_out, k))
    if bias is not None and (bias.shape != (n_out,) or bias.dtype != x.dtype or bias.device != x.device or
                             not bias.is_contiguous()):
        raise ValueError("contiguous bias [%d] in the type and on the device of x expected" % n_out)
    dev = x.device
    ldy = n_out
    if out is None:
        y = torch.empty((n, n_out), dtype=x.dtype, device=dev)
    else:
        y, ldy = out, _rows(out, "out", n_out, dev, x.dtype)
        if y.shape[0] != n or ldy < n_out:
            raise ValueError("out [%d, %d] with rows of its own expected" % (n, n_out))
    low = torch.empty((n, r), dtype=torch.float32, device=dev) if keep_low else None
    if n:
        work = torch.empty(size_of("flm_adapter_workspace", n, k, n_out, r, e, DTYPES[x.dtype]), dtype=torch.uint8, device=dev)
        launch(dev, "flm_adapter_linear", x.data_ptr(), ldx, weight.data_ptr(), ldw, bias.data_ptr() if bias is not None else None,
               a.data_ptr(), b.data_ptr(), groups.buf.data_ptr(), *scales, n, k, n_out, r, e, DTYPES[x.dtype], work.data_ptr(),
               y.data_ptr(), ldy, low.data_ptr() if keep_low else None)
    return (y, low) if keep_low else y


def adapter_linear_backward(dy, x, weight, a, b, groups, low, scale=1.0, need_dx=True, da=None, db=None):
    """Gradients (dx, da, db) of adapter_linear for the gradient dy [n, N] of y; the shared projection is held fixed.
    low: what adapter_linear kept.  need_dx = False: dx is None and weight is not read (None is taken).  da, db: contiguous
    tensors like a and b that receive the gradients (fresh ones by default; they share no element with an input); adapters
    without rows get zeros."""
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


class NetworkAdapters:
    """Low-rank adapters of a Dueling_DQN's two first dense layers (98 % of its weights), n_adapters of them: the network is
    shared, a map (or whatever an id stands for) owns (a, b) of either layer.  All parameters are one flat float32 buffer;
    a starts uniform within 1/sqrt(inputs), b as zeros, so that a new adapter changes nothing.  scale = alpha / rank
    (alpha None: 1)."""

    PARTS = ("a_adv", "a_val", "b_adv", "b_val")

    def __init__(self, network, n_adapters, rank, alpha=None):
        n_adapters, rank = int(n_adapters), int(rank)
        if not 1 <= n_adapters <= GROUPS_MAX or not 1 <= rank <= ADAPTER_MAX_RANK:
            raise ValueError("1..%d adapters of rank 1..%d" % (GROUPS_MAX, ADAPTER_MAX_RANK))
        self._allocate(network, n_adapters, rank, 1.0 if alpha is None else float(alpha) / rank)
        for a in (self.a_adv, self.a_val):
            a.uniform_(-self.inputs ** -0.5, self.inputs ** -0.5)

    def _allocate(self, network, n_adapters, rank, scale):
        self.n_adapters, self.rank, self.scale = n_adapters, rank, scale
        self.inputs, self.outputs = network.fc1_adv.in_features, network.fc1_adv.out_features
        self.device = network.flat_params().device
        self.flat = torch.zeros(sum(n for _, n in self._layout()), dtype=torch.float32, device=self.device)
        self.__dict__.update(self.views(self.flat))

    def _layout(self):
        e, r, k, n = self.n_adapters, self.rank, self.inputs, self.outputs
        return [((e, r, k), e * r * k), ((e, r, k), e * r * k), ((e, n, r), e * n * r), ((e, n, r), e * n * r)]

    def views(self, flat):
        """The four parameters (or their gradients, in a buffer of the same layout) by name."""
        out, at = {}, 0
        for name, (shape, n) in zip(self.PARTS, self._layout()):
            out[name] = flat[at:at + n].view(shape)
            at += n
        return out

    def state_dict(self):
        return {name: getattr(self, name).clone() for name in self.PARTS}

    def check_state_dict(self, state):
        """Whether load_state_dict() takes this; raises if not."""
        for name in self.PARTS:
            if tuple(state[name].shape) != tuple(getattr(self, name).shape):
                raise ValueError("%s %s expected" % (name, tuple(getattr(self, name).shape)))

    def load_state_dict(self, state):
        self.check_state_dict(state)
        for name in self.PARTS:
            getattr(self, name).copy_(state[name])

    def copy_for(self, network):
        """The same adapters, values and scale, beside another network of the same shape (the target network)."""
        other = object.__new__(type(self))
        other._allocate(network, self.n_adapters, self.rank, self.scale)
        other.flat.copy_(self.flat)
        return other

    def q_values(self, network, obs_u8, plane_stride, groups, out=None, features=None, keep=False):
        """Q-values [n, actions] of uint8 observations [n, 3, plane_stride] with the adapters of groups = group_rows(ids,
        n_adapters), ids the adapter of each observation; observations without one get the network's own values.  All rails
        are computed.  out: a float32 buffer of at least n * actions floats, whose first the result is; features: one of n * inputs
        floats (both optional, of any shape).
        keep: returns (q, what gradients() takes)."""
        if network.height % 3:
            raise ValueError("observations have three planes: the network height must be 3*max_rails")
        n = obs_u8.shape[0]
        if obs_u8.dtype != torch.uint8 or tuple(obs_u8.shape[1:]) != (3, plane_stride) or not obs_u8.is_contiguous():
            raise ValueError("contiguous uint8 observations [n, 3, plane_stride] expected")
        flat = network.flat_params()
        if obs_u8.device != flat.device:
            raise ValueError("observations on the network's device expected")
        for name, t, want in (("out", out, n * network.action_space), ("features", features, n * self.inputs)):
            if t is not None and (t.dtype != torch.float32 or t.device != flat.device or not t.is_contiguous() or t.numel() < want):
                raise ValueError("%s: a contiguous float32 buffer of at least %d elements on the network's device expected" % (name, want))
        q = torch.empty((n, network.action_space), dtype=torch.float32, device=flat.device) if out is None else \
            out.view(-1)[:n * network.action_space].view(n, network.action_space)
        x = torch.empty(n * self.inputs, dtype=torch.float32, device=flat.device) if features is None else features.view(-1)
        x = x[:n * self.inputs].view(n, self.inputs)
        hidden = torch.empty((n, 2 * self.outputs), dtype=torch.float32, device=flat.device)
        half = self.outputs
        if n:
            launch(flat.device, "flm_dqn_features_u8", flat.data_ptr(), obs_u8.data_ptr(), n, network.height // 3, network.width,
                   int(plane_stride), network.action_space, x.data_ptr())
        res = [adapter_linear(x, layer.weight.data, layer.bias.data, a, b, groups, scale=self.scale, keep_low=keep, out=y)
               for layer, a, b, y in ((network.fc1_adv, self.a_adv, self.b_adv, hidden[:, :half]),
                                      (network.fc1_val, self.a_val, self.b_val, hidden[:, half:]))]
        if n:
            launch(flat.device, "flm_dqn_heads", flat.data_ptr(), hidden.data_ptr(), n, network.height, network.width,
                   network.action_space, q.data_ptr())
        if not keep:
            return q
        return q, (x, hidden, groups, res[0][1], res[1][1])

    def gradients(self, kept, dhidden, grads):
        """The adapters' gradients from the gradient dhidden [n, 1024] of the layers' pre-activations, into the flat buffer
        grads; kept: from q_values."""
        x, _, groups, low_adv, low_val = kept
        into, half = self.views(grads), self.outputs
        for dy, low, part in ((dhidden[:, :half], low_adv, "adv"), (dhidden[:, half:], low_val, "val")):
            adapter_linear_backward(dy, x, None, getattr(self, "a_" + part), getattr(self, "b_" + part), groups, low, scale=self.scale,
                                    need_dx=False, da=into["a_" + part], db=into["b_" + part])


class AdapterAdam:
    """torch.optim.Adam (default options) over the flat parameters of a NetworkAdapters (flm_dqn_adam).  An adapter without
    rows in a step has a zero gradient; its moments decay and move it as Adam's do."""

    def __init__(self, adapters, lr, betas=(0.9, 0.999), eps=1e-8):
        self.adapters, self.lr, self.betas, self.eps = adapters, lr, betas, eps
        self.m, self.v, self.grads = (torch.zeros_like(adapters.flat) for _ in range(3))
        self.step_count = 0

    def state_dict(self):
        return {"m": self.m.clone(), "v": self.v.clone(), "step_count": self.step_count}

    def check_state_dict(self, state):
        """Whether load_state_dict() takes this; raises if not."""
        if state is not None and (not state["m"].shape == state["v"].shape == self.m.shape or int(state["step_count"]) < 0):
            raise ValueError("moments of %d adapter parameters expected" % self.m.numel())

    def load_state_dict(self, state):
        """None: as before the first step."""
        self.check_state_dict(state)
        for name in ("m", "v"):
            getattr(self, name).zero_() if state is None else getattr(self, name).copy_(state[name])
        self.step_count = 0 if state is None else int(state["step_count"])

    def step(self, target=None, tau=None):
        """One step with self.grads; with target (the target's NetworkAdapters) and tau its soft update in the same pass."""
        self.step_count += 1
        p = self.adapters.flat
        args = [t.data_ptr() for t in (p, self.grads, self.m, self.v)]
        hyper = (float(self.lr), float(self.betas[0]), float(self.betas[1]), float(self.eps), self.step_count)
        if target is None:
            launch(p.device, "flm_dqn_adam", *args, p.numel(), *hyper)
        else:
            launch(p.device, "flm_dqn_adam_soft_update", *args, target.flat.data_ptr(), p.numel(), *hyper, float(tau))
