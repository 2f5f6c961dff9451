"""What the AdamW step and the gradient clip refuse, count and remember, on the CPU."""
import ctypes as C

import pytest
import torch

import came_b200
from came_b200 import _host, _lib


def test_clip_refuses_addresses_off_their_elements():
    """(the kernels take 16 bytes from the first boundary of an element on)"""
    lib = _lib.load()
    need = lib.came_b200_clip_workspace_bytes(1)

    def code(at, dtype, norm=0x1000, n=100):
        return lib.came_b200_clip_grad_norm((_lib.CameGradRef * 1)(_lib.CameGradRef(at, n, dtype, 0)), 1, 1.0, norm, 0x2000, need, None)

    for at, dtype in ((0x10001, _lib.DT_F32), (0x10002, _lib.DT_F32), (0x10001, _lib.DT_F16), (0x10003, _lib.DT_BF16)):
        assert code(at, dtype) == _lib.E_INVALID and b"aligned" in lib.came_b200_last_error()
    assert code(0x10000, _lib.DT_F32, norm=0x1002) == _lib.E_INVALID and b"aligned" in lib.came_b200_last_error()
