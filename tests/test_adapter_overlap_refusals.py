"""Results of the adapter calls that share memory with an input or with each other, beside the matrices.  No GPU: every call is
refused before a launch."""
import ctypes

import pytest

from flatland_marl_amd import _lib

at = ctypes.c_void_p
n, K, N, r, E = 8, 64, 32, 4, 2


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_forward(dtype, size):
    lib = _lib.load()
    ok = [at(0x100000), K, at(0x200000), K, at(0x280000), at(0x300000), at(0x400000), at(0x500000), at(0x580000), 1.0, n, K, N, r, E,
          dtype, at(0x600000), at(0x700000), N, at(0x800000), None]
    y_bytes, low_bytes = n * N * size, n * r * 4
    ints = lib.flm_group_rows_ints(n, E)
    inputs = {0: n * K * size, 2: N * K * size, 4: N * size, 5: E * r * K * size, 6: E * N * r * size, 7: 4 * ints, 8: 4 * E}
    for i, bytes_of in inputs.items():
        for out, own in ((17, y_bytes), (19, low_bytes)):
            for place in (ok[i].value, ok[i].value + bytes_of - 4, ok[i].value - own + 4):
                args = list(ok)
                args[out] = at(place)
                assert lib.flm_adapter_linear(*args) == -4, (i, out, place)
    for place in (ok[17].value, ok[17].value + y_bytes - 4, ok[17].value - low_bytes + 4):
        args = list(ok)
        args[19] = at(place)
        assert lib.flm_adapter_linear(*args) == -4, place


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_backward(dtype, size):
    lib = _lib.load()
    ok = [at(0x100000), N, at(0x200000), K, at(0x300000), K, at(0x400000), at(0x500000), at(0x580000), at(0x5c0000), 1.0, at(0x600000),
          n, K, N, r, E, dtype, at(0x680000), at(0x700000), K, at(0x800000), at(0x900000), None]
    ints = lib.flm_group_rows_ints(n, E)
    outs = {19: n * K * size, 21: E * r * K * size, 22: E * N * r * size}
    for out, own in outs.items():
        for i, bytes_of in ((8, 4 * ints), (9, 4 * E), (11, 4 * n * r)):
            for place in (ok[i].value, ok[i].value + bytes_of - 4, ok[i].value - own + 4):
                args = list(ok)
                args[out] = at(place)
                assert lib.flm_adapter_linear_backward(*args) == -4, (i, out, place)
