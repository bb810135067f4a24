"""What flm_grad_clip refuses beside its sizes: memory that tensors share, pointers between elements.  No GPU: every call here
is refused before a launch."""
import ctypes

import pytest

from flatland_marl_amd import _lib

P = ctypes.c_void_p(4096)
N = 64                                                       # elements of every tensor


def _clip(src, dst, kinds=None, numel=None, workspace=P, norm=P):
    n = len(src)
    return _lib.load().flm_grad_clip((ctypes.c_void_p * n)(*src), None if dst is None else (ctypes.c_void_p * n)(*dst),
                                     (ctypes.c_int64 * n)(*(numel or [N] * n)), (ctypes.c_int32 * n)(*(kinds or [0] * n)), n, 1.0, 0,
                                     workspace, norm, None)


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("shift", [0, 4, -4, 4 * (N - 1), -4 * (N - 1)])
def test_a_tensor_that_only_counts_is_not_written_over(shift, order):
    """src {p, q}: p counts in the norm alone; q's result, in place or elsewhere, must not reach p."""
    p, q, far = 0x100000, 0x200000, 0x300000
    for src, dst in (([p, q], [None, p + shift]), ([p, p + shift], [None, p + shift])):
        assert _clip([src[i] for i in order], [dst[i] for i in order]) == -4
    # a span that begins far below and reaches over both, behind one that ends early
    assert _clip([p - 4 * N, p, far], [None, None, p - 4 * 3 * N], numel=[N, 1, 4 * N]) == -4


def test_spans_inside_others():
    """An overlap that is not between neighbours in the order of addresses."""
    p, far = 0x100000, 0x300000
    # two that only count, the first of which reaches over the third's result
    assert _clip([p, p + 8, far], [None, None, p + 800], numel=[1000, 2, 4]) == -4
    # a source clipped elsewhere that reaches over another
    assert _clip([p, p + 8, p + 800], [far, None, far + 0x100000], numel=[1000, 2, 4]) == -4


@pytest.mark.parametrize("kind,off", [(0, 1), (0, 2), (0, 3), (1, 1), (2, 1)])
def test_pointers_between_elements(kind, off):
    p, far = 0x100000, 0x300000
    assert _clip([p + off], [p + off], [kind]) == -1
    assert _clip([p], [far + off], [kind]) == -1
    assert _clip([p + off], None, [kind]) == -1
    assert _clip([p, p + 0x1000], [p, p + 0x1000 + off], [kind, kind]) == -1
    assert _clip([p], [p], [kind], workspace=ctypes.c_void_p(4100)) == -1
    assert _clip([p], [p], [kind], norm=ctypes.c_void_p(4098)) == -1
    ok = [ctypes.c_void_p(0x100000), 20, 31, 2, 8, 1, P, 1.0, 0, P, P, None]
    for i, at in ((0, 0x100000 + off), (6, 4096 + off), (9, 4100), (10, 4096 + off)):
        args = list(ok)
        args[i] = ctypes.c_void_p(at)
        assert _lib.load().flm_dqn_grad_clip(*args) == -1, i


def test_outputs_stay_with_their_gradients():
    """A None among the gradients and one among the outputs are not dropped apart from each other."""
    import torch
    from flatland_marl_amd import FlmError
    from flatland_marl_amd.gradients import clip_grad_norm_
    g, o = torch.ones(4), torch.zeros(4)
    with pytest.raises(ValueError):
        clip_grad_norm_([None, g], 1.0, out=[o, None])
    with pytest.raises(ValueError):
        clip_grad_norm_([g, g.clone()], 1.0, out=[o])
    for grads, out in (([None, g], [o, o]), ([None, g], [None, o]), ([None, g], [o]), (g, o), (iter([None, g]), iter([None, o])),
                       ([g], o)):
        with pytest.raises(FlmError):                       # (as far as the missing GPU)
            clip_grad_norm_(grads, 1.0, out=out)
    assert clip_grad_norm_([None], 1.0, out=[o]).item() == 0 and (o == 0).all()
    assert clip_grad_norm_([], 1.0, out=[o]).item() == 0 and clip_grad_norm_(iter(()), 1.0, out=iter(())).item() == 0
