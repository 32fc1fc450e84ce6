"""Argument checks of the 8-bit integer projections: every refusal comes back before any CUDA call."""
import ctypes

import pytest

# stand-ins for device pointers and for a pool; a refused call never reads through them
POINTER = 0x10000
POOL = ctypes.create_string_buffer(4096)


def linear(qm, pool=True, x=POINTER, x_scale=POINTER, weight=POINTER, weight_scale=POINTER, bias=0, residual=0, out=POINTER, rows=3,
           outer=8, inner=32):
    return qm.load_library().qm_linear_int8(ctypes.addressof(POOL) if pool else None, x, x_scale, weight, weight_scale, bias, residual,
                                            out, rows, outer, inner, None)


@pytest.mark.parametrize("change,text", [
    ({"pool": False}, b"pool is null"), ({"x": None}, b"null"), ({"x_scale": None}, b"null"), ({"weight": None}, b"null"),
    ({"weight_scale": None}, b"null"), ({"out": None}, b"null"), ({"rows": -1}, b"rows"), ({"outer": 0}, b"output width"),
    ({"inner": 0}, b"multiple of 16"), ({"inner": 24}, b"multiple of 16"), ({"inner": 65552}, b"65536"),
    ({"x": POINTER + 8}, b"aligned"), ({"weight": POINTER + 4}, b"aligned"), ({"out": POINTER + 2}, b"aligned"),
    ({"weight_scale": POINTER + 4}, b"aligned"), ({"bias": POINTER + 2}, b"aligned"), ({"residual": POINTER + 2}, b"aligned"),
    ({"x_scale": POINTER + 2}, b"aligned"),
])
def test_linear_refuses(qm, change, text):
    assert linear(qm, **change) == qm.QM_EINVAL
    assert text in qm.load_library().qm_last_error_string()


def test_no_rows_is_no_work(qm):
    assert linear(qm, rows=0, x=None, x_scale=None, out=None) == qm.QM_OK
    assert qm.load_library().qm_quantize_rows_int8(None, None, 1e-6, None, None, 0, 64, None) == qm.QM_OK


def test_gated_and_qkv_refuse(qm):
    lib = qm.load_library()
    p, pool = POINTER, ctypes.addressof(POOL)
    assert lib.qm_gate_up_swiglu_int8(pool, p, p, p, p, None, p, p, 3, 32, 64, None) == qm.QM_EINVAL
    assert lib.qm_gate_up_swiglu_int8(pool, p, p, p, p, p, None, p, 3, 32, 64, None) == qm.QM_EINVAL
    assert lib.qm_gate_up_swiglu_int8(pool, p, p, p, p, p, p + 4, p, 3, 32, 64, None) == qm.QM_EINVAL
    assert lib.qm_gate_up_swiglu_int8(None, p, p, p, p, p, p, p, 3, 32, 64, None) == qm.QM_EINVAL
    assert lib.qm_qkv_linear_int8(pool, p, p, p, p, None, p, p, None, p, None, None, p, p, p, 3, 32, 16, 8, None) == qm.QM_EINVAL
    assert lib.qm_qkv_linear_int8(pool, p, p, p, p, None, p, p, None, p, p, None, p, p, p, 3, 32, 16, 0, None) == qm.QM_EINVAL


def test_quantiser_refuses(qm):
    lib = qm.load_library()
    p = POINTER
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, p, -1, 64, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, p, 1, 0, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, p, 1, 24577, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(None, None, 1e-6, p, p, 1, 64, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, None, p, 1, 64, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, None, 1, 64, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p + 1, None, 1e-6, p, p, 1, 64, None) == qm.QM_EINVAL
    assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, p + 2, 1, 64, None) == qm.QM_EINVAL


def test_a_row_number_past_the_last_tile_would_not_fit_an_int(qm):
    lib, p = qm.load_library(), POINTER
    for rows in (2 ** 31 - 1, 2 ** 31 - 255):
        assert linear(qm, outer=rows) == qm.QM_EINVAL and b"output width" in lib.qm_last_error_string()
        assert linear(qm, rows=rows) == qm.QM_EINVAL and b"rows" in lib.qm_last_error_string()
        assert lib.qm_quantize_rows_int8(p, None, 1e-6, p, p, rows, 64, None) == qm.QM_EINVAL
