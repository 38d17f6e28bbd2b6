"""The far ends of what the decoder operators' C entries admit: host checks, no GPU."""
import ctypes

from backtoreality_amd.pointnet2 import _ext

lib = _ext._lib
PTR = 4096   # a non-null address for entries that refuse before they read anything


def _error():
    return lib.btr_last_error().decode()


def _attention(**kw):
    p = _ext.CrossAttention(dtype=1, b=2, lq=3, lk=70, h=4, hk=2, d=64, q=PTR, k=PTR, v=PTR, scale=0.125)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def test_attention_grids_beyond_32_bits_are_refused():
    """A workgroup per batch entry, key head and tile: thread numbers of 32 bits."""
    for dtype in (0, 1, 2):
        for sizes in (dict(b=2 ** 24, lq=1, lk=1, h=1, hk=1), dict(b=2 ** 21, lq=1, lk=1, h=8, hk=8),
                      dict(b=2 ** 14, lq=2 ** 16, lk=1), dict(b=2 ** 14, lq=2 ** 16, lk=1, d=128)):
            p = _attention(dtype=dtype, **sizes)
            at = ctypes.addressof(p)
            assert lib.btr_cross_attention_fwd_workspace_bytes(at) == 0
            assert "too many" in _error(), sizes
            assert lib.btr_cross_attention_bwd_workspace_bytes(at, PTR) == 0
            assert lib.btr_cross_attention_fwd(at, PTR, None, PTR, 1 << 62, None) == -1
            assert lib.btr_cross_attention_bwd(at, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 1 << 62, None) == -1
        # the keys' workgroups are the backward's alone
        p = _attention(dtype=dtype, b=2 ** 12, lq=1, lk=2 ** 19, d=8)
        at = ctypes.addressof(p)
        assert lib.btr_cross_attention_bwd_workspace_bytes(at, PTR) == 0 and "too many" in _error()
        assert lib.btr_cross_attention_bwd(at, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 1 << 62, None) == -1
        # the largest batch that has room
        p = _attention(dtype=dtype, b=2 ** 24 - 1, lq=1, lk=1, h=1, hk=1, d=8)
        assert lib.btr_cross_attention_bwd_workspace_bytes(ctypes.addressof(p), PTR) > 0


def test_linear_grids_beyond_32_bits_are_refused():
    for sizes in (dict(m=2 ** 30, n=512, k=8), dict(m=2 ** 30, n=8, k=512)):
        p = _ext.Linear(dtype=1, act=0, x=PTR, weight=PTR, ldx=2 ** 10, ldw=2 ** 10, **sizes)
        assert lib.btr_linear_fwd(ctypes.addressof(p), PTR, None, PTR, 1 << 60, None) == -1
        assert "linear_fwd" in _error()


def test_workspaces_off_a_16_byte_boundary_are_refused():
    odd = PTR + 8
    p = _attention(lq=1, lk=100000)
    need = lib.btr_cross_attention_fwd_workspace_bytes(ctypes.addressof(p))
    assert need > 0
    assert lib.btr_cross_attention_fwd(ctypes.addressof(p), PTR, None, odd, need, None) == -1
    assert "16-byte" in _error()
    assert lib.btr_cross_attention_bwd(ctypes.addressof(p), PTR, PTR, PTR, PTR, PTR, PTR, odd, 1 << 40,
                                       None) == -1 and "16-byte" in _error()
    p = _ext.Linear(dtype=1, m=100, n=100, k=15, act=0, x=PTR, weight=PTR, ldx=15, ldw=15)
    need = lib.btr_linear_fwd_workspace_bytes(ctypes.addressof(p))
    assert lib.btr_linear_fwd(ctypes.addressof(p), PTR, None, odd, need, None) == -1
    assert "16-byte" in _error()
    assert lib.btr_linear_bwd(ctypes.addressof(p), None, PTR, 100, PTR, PTR, PTR, odd, 1 << 40,
                              None) == -1 and "16-byte" in _error()
