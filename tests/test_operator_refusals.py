"""What the adapter and gradient calls refuse, checked without a GPU: the C entry points' own checks, and the Python
layer's (on CPU tensors it never gets as far as a launch)."""
import ctypes

import pytest
import torch

from flatland_marl_amd import FlmError, _lib
from flatland_marl_amd.adapters import RowGroups, adapter_linear, group_rows
from flatland_marl_amd.gradients import _dense, clip_grad_norm_, grad_norm

P = ctypes.c_void_p(4096)                     # a pointer that is never followed: every call below is refused before a launch


def test_size_queries():
    lib = _lib.load()
    assert lib.flm_group_rows_ints(0, 4) == 0 and lib.flm_group_rows_ints(10, 0) == 0
    # order and key padded to 12, twice four offsets, tiles of 32 rows: one full tile's worth and one per group
    assert lib.flm_group_rows_ints(10, 3) == 12 + 12 + 4 + 4 + 2 * (1 + 3)
    assert lib.flm_group_rows_workspace(8192, 100) == 0 and lib.flm_group_rows_workspace(8193, 100) >= 101
    for n, k, n_out, r, e in ((0, 8, 8, 4, 1), (8, 0, 8, 4, 1), (8, 8, 8, 0, 1), (8, 8, 8, 129, 1), (8, 8, 8, 4, 2048),
                              (1 << 21, 8, 8, 4, 1)):
        assert lib.flm_adapter_workspace(n, k, n_out, r, e, 0) == 0
        assert lib.flm_adapter_backward_workspace(n, k, n_out, r, e, 0, 1) == 0
    assert lib.flm_adapter_workspace(8, 64, 32, 4, 1, 2) > 0
    assert lib.flm_adapter_backward_workspace(8, 64, 32, 4, 1, 3, 1) == 0


def test_group_rows_entry():
    lib = _lib.load()
    ok = [P, 0, 10, 3, P, None, None]
    for i, bad in ((0, None), (2, 0), (2, -5), (3, 0), (3, 2048), (4, None)):
        args = list(ok)
        args[i] = bad
        assert lib.flm_group_rows(*args) == -1, i
    assert lib.flm_group_rows(P, 0, 8193, 3, P, None, None) == -1              # needs a workspace
    for i, at in ((0, 4098), (4, 4104)):                                       # an int, sixteen bytes
        args = list(ok)
        args[i] = ctypes.c_void_p(at)
        assert lib.flm_group_rows(*args) == -1, i
    assert lib.flm_group_rows(ctypes.c_void_p(4100), 1, 10, 3, P, None, None) == -1


def test_adapter_entries():
    lib = _lib.load()
    ok = [P, 64, P, 64, None, P, P, P, None, 1.0, 8, 64, 32, 4, 2, 1, P, P, 32, None, None]
    for i, bad in ((0, None), (1, -1), (2, None), (3, -2), (5, None), (6, None), (7, None), (10, 0), (10, (1 << 20) + 1), (11, 0),
                   (12, 0), (13, 0), (13, 129), (14, 0), (14, 2048), (15, -1), (15, 3), (16, None), (16, ctypes.c_void_p(4100)),
                   (17, None), (18, 31)):
        args = list(ok)
        args[i] = bad
        assert lib.flm_adapter_linear(*args) == -1, i
    ok = [P, 32, P, 64, P, 64, P, P, P, None, 1.0, P, 8, 64, 32, 4, 2, 1, P, P, 64, P, P, None]
    for i, bad in ((0, None), (1, -1), (2, None), (3, -1), (4, None), (5, -1), (6, None), (7, None), (8, None), (11, None), (12, 0),
                   (15, 200), (17, 5), (18, None), (18, ctypes.c_void_p(8)), (20, 63), (21, None), (22, None)):
        args = list(ok)
        args[i] = bad
        assert lib.flm_adapter_linear_backward(*args) == -1, i


def test_adapter_operands_between_elements():
    lib = _lib.load()
    fwd = [P, 64, P, 64, P, P, P, P, P, 1.0, 8, 64, 32, 4, 2, 1, P, P, 32, P, None]
    bwd = [P, 32, P, 64, P, 64, P, P, P, P, 1.0, P, 8, 64, 32, 4, 2, 1, P, P, 64, P, P, None]
    for call, ok, places in ((lib.flm_adapter_linear, fwd, ((0, 1), (2, 1), (4, 1), (5, 1), (6, 1), (7, 8), (8, 2), (17, 1), (19, 2))),
                             (lib.flm_adapter_linear_backward, bwd, ((0, 1), (2, 1), (4, 1), (6, 1), (7, 1), (8, 8), (9, 2), (11, 2),
                                                                     (19, 1), (21, 1), (22, 1)))):
        for i, off in places:
            args = list(ok)
            args[i] = ctypes.c_void_p(4096 + off)
            assert call(*args) == -1, i


def test_adapter_results_that_share_memory():
    """Host addresses only: every call is refused before a launch.  n 8, K 64, N 32, r 4, E 2, bf16."""
    lib = _lib.load()
    at = ctypes.c_void_p
    ok = [at(0x100000), 64, at(0x200000), 64, at(0x280000), at(0x300000), at(0x400000), P, None, 1.0, 8, 64, 32, 4, 2, 1, P, at(0x500000),
          32, None, None]
    sizes = {0: 8 * 64, 2: 32 * 64, 4: 32, 5: 2 * 4 * 64, 6: 2 * 32 * 4}          # elements of each input
    for i, n in sizes.items():
        for y in (ok[i].value, ok[i].value + 2 * n - 2, ok[i].value - 2 * 8 * 32 + 2):
            args = list(ok)
            args[17] = at(y)
            assert lib.flm_adapter_linear(*args) == -4, (i, y)
    # columns of one matrix: x and y share 16 of them
    args = list(ok)
    args[1], args[17], args[18] = 96, at(0x100000 + 2 * 48), 96
    assert lib.flm_adapter_linear(*args) == -4
    args[17] = at(0x100000 + 2 * 64 + 2 * 2)                                      # runs over into x's next row
    assert lib.flm_adapter_linear(*args) == -4
    ok = [at(0x100000), 32, at(0x200000), 64, at(0x300000), 64, at(0x400000), at(0x500000), P, None, 1.0, at(0x600000), 8, 64, 32, 4, 2, 1, P,
          at(0x700000), 64, at(0x800000), at(0x900000), None]
    for out in (19, 21, 22):
        for other in (0, 2, 4, 6, 7, 11, 19, 21, 22):
            if out != other:
                args = list(ok)
                args[out] = ok[other]
                assert lib.flm_adapter_linear_backward(*args) == -4, (out, other)


def test_gradient_entries():
    lib = _lib.load()
    src = (ctypes.c_void_p * 2)(4096, 8192)
    numel, kinds = (ctypes.c_int64 * 2)(5, 6), (ctypes.c_int32 * 2)(0, 1)
    ok = [src, src, numel, kinds, 2, 1.0, 0, P, P, None]
    for i, bad in ((0, None), (2, None), (3, None), (4, 0), (4, 65537), (5, -1.0), (5, float("nan")), (7, None), (8, None)):
        args = list(ok)
        args[i] = bad
        assert lib.flm_grad_clip(*args) == -1, i
    for bad_numel, bad_kind, bad_src in (((5, -1), (0, 0), (4096, 8192)), ((5, 6), (0, 3), (4096, 8192)), ((5, 6), (0, 0), (4096, None))):
        assert lib.flm_grad_clip((ctypes.c_void_p * 2)(*bad_src), src, (ctypes.c_int64 * 2)(*bad_numel),
                                 (ctypes.c_int32 * 2)(*bad_kind), 2, 1.0, 0, P, P, None) == -1
    # memory shared between tensors that are written
    for a, b in (((4096, 4100), None), ((4096, 4096), None), ((4096, 8192), (8200, 20480)), ((4096, 8192), (16384, 16392))):
        src = (ctypes.c_void_p * 2)(*a)
        dst = (ctypes.c_void_p * 2)(*(b or a))
        assert lib.flm_grad_clip(src, dst, numel, kinds, 2, 1.0, 0, P, P, None) == -4
    ok = [P, 20, 31, 2, 8, 1, P, 1.0, 0, P, P, None]
    for i, bad in ((0, None), (1, 0), (2, 0), (3, 0), (3, 17), (4, 21), (4, -1), (4, 0), (5, 0), (6, None), (7, -1.0), (9, None), (10, None)):
        args = list(ok)
        args[i] = bad
        assert lib.flm_dqn_grad_clip(*args) == -1, i


def test_python_layer():
    f = torch.zeros
    with pytest.raises(FlmError):
        group_rows(f(4, dtype=torch.int32), 3)
    for ids, e in ((f(2, 2, dtype=torch.int32), 3), (f(4), 3), (f(4, dtype=torch.int32), 0), (f(4, dtype=torch.int32), 2048)):
        with pytest.raises(ValueError):
            group_rows(ids, e)
    g = RowGroups(f(20, dtype=torch.int32), 4, 2)
    with pytest.raises(FlmError):
        adapter_linear(f(4, 8), f(6, 8), None, f(2, 3, 8), f(2, 6, 3), g)
    with pytest.raises(ValueError):
        adapter_linear(f(4, 8, dtype=torch.float64), f(6, 8), None, f(2, 3, 8), f(2, 6, 3), g)
    for bad in ([f(4)], f(4)):
        with pytest.raises(FlmError):
            clip_grad_norm_(bad, 1.0)
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, norm_type=1.0)):
        with pytest.raises(ValueError):
            clip_grad_norm_([f(4)], **kw)
    with pytest.raises(ValueError):
        grad_norm([], norm_type=3)
    assert _dense(f(3, 4)) and _dense(f(3, 4).t()) and _dense(f(0)) and _dense(f(2, 3, 4, 5).permute(0, 3, 1, 2))
    assert not _dense(f(3, 4)[:, :2]) and not _dense(f(1, 4).expand(3, 4)) and not _dense(f(8)[::2])
