"""Head strides that the attention over packed rows takes: below 2^29 over all heads, whatever the number of heads.  Nothing is
launched: the calls end at a missing workspace."""

import ctypes

import pytest

from cqgdn import _lib


@pytest.mark.parametrize("heads,stride,taken", [
    (31, 17318416, True),  # 31 strides are 16 below 2^29
    (31, 17318424, False), (1, (1 << 29) - 8, True), (1, 1 << 29, False), (2, 1 << 28, False), (2, (1 << 28) - 8, True),
    (7, 76695848, False), (3, 1 << 62, False),
])
def test_head_strides_up_to_their_limit(heads, stride, taken):
    lib = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    T, S = 100, 5000
    assert lib.cqgdn_attend_fwd_workspace_size(T, S, heads, heads, 64) > 0
    for name in ("qh", "kh", "vh"):
        a = dict(q=p, qt=64, qh=64, k=p, kt=64, kh=64, v=p, vt=64, vh=64, dtype=0, T=T, S=S, heads=heads, kv=heads, D=64, first=None,
                 limit=p, positions=None, scale=1.0, cap=0.0, slopes=None, out=p, lse=p, ws=None, n=0, stream=None)
        a[name] = stride
        assert lib.cqgdn_attend_fwd(*a.values()) == _lib.EINVAL
        assert (b"workspace" in lib.cqgdn_last_error()) == taken, lib.cqgdn_last_error()
