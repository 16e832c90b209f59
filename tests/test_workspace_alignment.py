"""Workspaces that are not aligned as documented are refused before a launch (on the CPU: nothing gets that far)."""
import ctypes

import pytest

from rgd_triton_amd import _hip

D4 = (0x1000, 4096, 64, 64)
WORKSPACE = -4


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_decode_workspace(off):
    args = _hip.decode_args(1, 4, 2, 64, *D4, *D4, *D4, *D4, 8, 16, 0x1000, 4, 4, 0x1000, 0, 0, 0, 0, 0, 0, 0, 0x1000 + off, 1 << 30, 0, 2, 0.125)
    assert _hip.lib().rgd_paged_decode(args, None) == WORKSPACE and b"aligned" in _hip.lib().rgd_last_error()


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_bias_workspaces(off):
    lib = _hip.lib()
    starts, buckets = (ctypes.c_int32 * 3)(-5, 0, 3), (ctypes.c_int32 * 3)(2, 1, 0)
    buf, work = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1000 + off)
    t4 = _hip.desc4(*D4)
    assert lib.rgd_rel_bias_bwd(2, 4, 4, t4, 0, 3, starts, buckets, 0, buf, 2, 3, 0, work, 1 << 20, None) == WORKSPACE
    assert b"aligned" in lib.rgd_last_error()
    # the forward uses one for large matrices only
    assert lib.rgd_rel_bias_fwd_workspace(8, 4096, 4096, 2) > 0
    assert lib.rgd_rel_bias_fwd(8, 4096, 4096, buf, 8, 3, 0, 3, starts, buckets, 0, t4, 2, work, 1 << 30, None) == WORKSPACE
    assert b"aligned" in lib.rgd_last_error()
