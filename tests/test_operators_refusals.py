"""Arguments of the operators' C entries that have to be refused before any launch, on a host without a GPU."""
import ctypes

import pytest

from ra_spmm import capi

OK, INVALID, UNSUPPORTED = 0, 1, 4


def norm(**kw):
    s = capi.NormShape(rows=3, q_heads=4, k_heads=2, head_dim=16, rot_dim=8, positions=10, layout=0, dtype=0, eps=1e-6,
                       ldq=64, ldk=32)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("positions", [0, -1])
def test_rotation_by_an_empty_table(positions):
    """No row of the table may be read, so none may be asked for."""
    lib, fake, n = capi.load(), ctypes.c_void_p(4096), ctypes.c_int64()
    s = norm(positions=positions)
    assert lib.ra_head_norm(ctypes.byref(s), *[fake] * 8, None) == INVALID and b"table" in lib.ra_last_error()
    assert lib.ra_head_norm_backward(ctypes.byref(s), *[fake] * 13, 1 << 30, None) == INVALID
    assert b"table" in lib.ra_last_error()
    # Nothing to read without rows or without a rotation.
    assert lib.ra_head_norm(ctypes.byref(norm(positions=positions, rows=0)), *[fake] * 8, None) == OK
    assert lib.ra_head_norm_workspace(ctypes.byref(norm(positions=positions, rot_dim=0)), ctypes.byref(n)) == OK
