"""Argument checks of the shared-prefix attention: every refusal comes back before any CUDA call."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
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


def test_the_tensors_of_an_empty_batch_may_be_null(qm):
    """An empty PyTorch tensor has no address."""
    assert shared(qm, batch=0, q=None, lens=None, table=None, out=None, starts=None, pages=None, groups=0) == qm.QM_OK
    assert shared(qm, batch=0, q=None, lens=None, table=None, out=None) == qm.QM_OK
    assert shared(qm, batch=0, layer=2, q=None) == qm.QM_EINVAL


def test_workspace_covers_the_plain_call_and_the_pieces(qm):
    lib = qm.load_library()
    pool = ctypes.addressof(POOL)
    assert lib.qm_decode_shared_workspace_bytes(None, 4) == 0
    for batch in (1, 64, 256):
        need = lib.qm_decode_shared_workspace_bytes(pool, batch)
        assert need >= lib.qm_decode_workspace_bytes(batch, 8) + 2 * 148 * 128 * 520


class Tensor:
    """What the Python call looks at in a tensor."""

    def __init__(self, dtype, *shape, device=0):
        self.dtype, self.shape, self.device = dtype, shape, device

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return True

    def numel(self):
        return 1 << 30

    def data_ptr(self):
        return P

    def stride(self):
        return ()


class Library:
    """Counts the workspaces it is asked to prepare; `init` and `launch` are what those calls answer."""

    def __init__(self, init, launch):
        self.prepared, self.init, self.launch = 0, init, launch

    def qm_decode_shared_workspace_bytes(self, pool, batch):
        return 64

    def qm_decode_workspace_init(self, workspace, size, stream):
        self.prepared += 1
        return self.init

    def qm_decode_attention_shared(self, *args):
        return self.launch


def python_call(qm, monkeypatch, library, pool_device=0, device=0, seq_lens=3):
    import torch

    monkeypatch.setattr(torch.cuda, "current_device", lambda: device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch, "empty", lambda *size, **kw: Tensor(torch.uint8, device=device))
    monkeypatch.setattr(qm, "_stream", lambda: 0)
    eng = object.__new__(qm.TalkerAttention)
    eng.lib, eng.pool, eng.q_heads, eng.kv_heads, eng._shared_workspace = library, None, 4, 2, None
    eng.rope_cos = Tensor(torch.bfloat16, 1, 128, device=pool_device)
    bf16, i32 = torch.bfloat16, torch.int32

    def call():
        q = Tensor(bf16, 3, 4, 128, device=device)
        return eng.launch_attention_shared(0, q, Tensor(i32, seq_lens, device=device), Tensor(i32, 3, 5, device=device),
                                           Tensor(i32, 2, device=device), Tensor(i32, 1, device=device), 2, out=q)
    return eng, call


def test_the_python_call_makes_its_workspace_once(qm, monkeypatch):
    library = Library(qm.QM_OK, qm.QM_OK)
    eng, call = python_call(qm, monkeypatch, library)
    call()
    first = eng._shared_workspace
    call()
    assert first is not None and eng._shared_workspace is first and library.prepared == 1


def test_a_call_from_another_device_leaves_no_workspace_there(qm, monkeypatch):
    """The pool is on device 0 and device 1 is current: later calls on device 0 must not be given memory of device 1."""
    library = Library(qm.QM_OK, qm.QM_EINVAL)
    eng, call = python_call(qm, monkeypatch, library, pool_device=0, device=1)
    with pytest.raises(qm.QmError):
        call()
    assert eng._shared_workspace is None and library.prepared == 0


def test_a_workspace_that_could_not_be_prepared_is_not_kept(qm, monkeypatch):
    library = Library(qm.QM_ECUDA, qm.QM_OK)
    eng, call = python_call(qm, monkeypatch, library)
    with pytest.raises(qm.QmError):
        call()
    assert eng._shared_workspace is None
    library.init = qm.QM_OK
    call()
    assert eng._shared_workspace is not None and library.prepared == 2


def test_the_mirror_frees_no_workspace_that_a_launch_was_given(tmp_path):
    """The C++ mirror with stand-ins for CUDA and the library, so that a workspace freed too early is seen on the CPU."""
    binary = tmp_path / "shared_workspace_test"
    toolkit = Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve().parent.parent
    cmd = ["g++", "-std=c++17", "-O1", "-I", str(toolkit / "include"), "-I", str(ROOT / "include"), "-I",
           str(ROOT / "qingming-qwen3-tts_b200" / "host"), str(ROOT / "tests" / "cpp" / "shared_workspace_test.cpp"), "-o", str(binary)]
    built = subprocess.run(cmd, capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0 and "SHARED_WORKSPACE_OK" in ran.stdout, ran.stdout + ran.stderr
