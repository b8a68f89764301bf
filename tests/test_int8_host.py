"""Host-side parts of the int8 and balance entry points that need no GPU: the descriptions' layout,
workspace sizes, and null arguments (each refused before anything touches a device)."""

import ctypes as C

import pytest

import vastloom_b200 as vb


def test_packed_descriptions_have_the_structures_layout():
    """The Python calls pack the descriptions as bytes: the same bytes as the structures."""
    ints = list(range(1, 16)), list(range(16, 20))
    d = vb._Int8LinearDesc(*ints[0], *ints[1], 2, 1, 0.5, 0)
    assert bytes(d) == vb._INT8_LINEAR_PACK(*ints[0], *ints[1], 2, 1, 0.5, 0)
    ints = list(range(1, 13)), list(range(13, 17))
    b = vb._BalanceDesc(*ints[0], *ints[1], 2, 1, 0.25, 0)
    assert bytes(b) == vb._BALANCE_PACK(*ints[0], *ints[1], 2, 1, 0.25, 0)


@pytest.mark.parametrize("rows,cols", [(0, 16), (1, 1), (7, 33), (4096, 4096), (1 << 20, 131071)])
def test_int8_workspace_holds_rows_and_scales(rows, cols):
    pitch = (cols + 15) // 16 * 16
    assert vb.int8_workspace_bytes(rows, cols) >= rows * pitch + rows * 4
    assert vb.int8_workspace_bytes(rows, cols) <= 2 * (rows * pitch + rows * 4) + 1024


@pytest.mark.parametrize("T,E,S", [(0, 1, 1), (1, 8, 1), (65536, 512, 1), (1000, 64, 1000), (65536, 256, 13)])
def test_balance_workspace_holds_every_sequence(T, E, S):
    n = vb.balance_workspace_bytes(T, E, S)
    assert S * (E + 1) * 4 <= n <= 1 << 30
    assert vb.balance_workspace_bytes(T, E, 0) == 0


def test_null_handles_are_errors():
    lib = vb.load_library()
    assert lib.vlb_int8_linear_device(None, None, None) == 1
    assert lib.vlb_int8_quantize_device(None, 0, None, 0, 0, None, None, 0.0, 1, 1, None, 0, None, None) == 1
    assert lib.vlb_int8_status(None, None) == 1
    assert lib.vlb_route_plan_device(None, None, None, 1, 1, 1, None, None, None, None, None, None) == 1
    assert lib.vlb_balance_loss_device(None, None, None) == 1
    buf = C.create_string_buffer(64)
    assert lib.vlb_last_error(None, buf, 64) == 0 and b"null handle" in buf.value
