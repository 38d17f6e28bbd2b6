"""The far ends of what the decoder operators' C entries admit: host checks, no GPU."""
import ctypes

from backtoreality_amd.pointnet2 import _ext

lib = _ext._lib
PTR = 4096   # a non-null address for entries that refuse before they read anything


def _error():
    return lib.btr_last_error().decode()


def test_linear_grids_beyond_32_bits_are_refused():
    for sizes in (dict(m=2 ** 30, n=512, k=8), dict(m=2 ** 30, n=8, k=512)):
        p = _ext.Linear(dtype=1, act=0, x=PTR, weight=PTR, ldx=2 ** 10, ldw=2 ** 10, **sizes)
        assert lib.btr_linear_fwd(ctypes.addressof(p), PTR, None, PTR, 1 << 60, None) == -1
        assert "linear_fwd" in _error()
