"""Argument checks of the shared-prefix attention: every refusal comes back before any CUDA call."""
import ctypes

import pytest

P = 0x10000


class Pool(ctypes.Structure):
    """The leading members of the library's pool object, as much of it as the checks read."""
    _fields_ = [("device", ctypes.c_int), ("layers", ctypes.c_int), ("num_pages", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("sm_count", ctypes.c_int), ("rest", ctypes.c_char * 256)]


POOL = Pool(0, 2, 10, 8, 148)


def shared(qm, pool=True, layer=0, q=P, lens=P, table=P, max_pages=4, batch=3, q_heads=16, starts=P, pages=P, groups=1, most=2, out=P, ws=P,
           ws_bytes=1 << 30):
    return qm.load_library().qm_decode_attention_shared(ctypes.addressof(POOL) if pool else None, layer, q, lens, table, max_pages, batch,
                                                        q_heads, starts, pages, groups, most, out, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    ({"pool": False}, "QM_EINVAL"), ({"layer": -1}, "QM_EINVAL"), ({"layer": 2}, "QM_EINVAL"), ({"q": None}, "QM_EINVAL"),
    ({"lens": None}, "QM_EINVAL"), ({"table": None}, "QM_EINVAL"), ({"out": None}, "QM_EINVAL"), ({"ws": None}, "QM_EINVAL"),
    ({"starts": None}, "QM_EINVAL"), ({"pages": None}, "QM_EINVAL"), ({"max_pages": 0}, "QM_EINVAL"), ({"batch": -1}, "QM_EINVAL"),
    ({"q_heads": 8}, "QM_EINVAL"), ({"groups": -1}, "QM_EINVAL"), ({"most": -1}, "QM_EINVAL"), ({"batch": 257}, "QM_ECAPACITY"),
    ({"groups": 257}, "QM_ECAPACITY"), ({"q": P + 8}, "QM_EINVAL"), ({"ws": P + 8}, "QM_EINVAL"), ({"ws_bytes": 100000}, "QM_EINVAL"),
])
def test_refusals(qm, change, code):
    assert shared(qm, **change) == getattr(qm, code)
    assert qm.load_library().qm_last_error_string()


def test_an_empty_batch_is_no_work(qm):
    assert shared(qm, batch=0) == qm.QM_OK


def test_workspace_covers_the_plain_call_and_the_pieces(qm):
    lib = qm.load_library()
    pool = ctypes.addressof(POOL)
    assert lib.qm_decode_shared_workspace_bytes(None, 4) == 0
    for batch in (1, 64, 256):
        need = lib.qm_decode_shared_workspace_bytes(pool, batch)
        assert need >= lib.qm_decode_workspace_bytes(batch, 8) + 2 * 148 * 128 * 520
