"""The 8-bit tape's operators on any machine: what they refuse at the ends of their ranges, and what their workspaces take."""
import ctypes as C

import pytest
import torch

from magnet_amd import _lib, ops


def test_widths_beyond_32_bits_are_refused():
    """a kernel counts columns in 32 bits"""
    wide = 2 ** 32 + 5
    meta = lambda *s, **k: torch.empty(*s, device="meta", **k)  # noqa: E731
    for W in (2 ** 31, wide):
        with pytest.raises(ValueError, match="columns"):
            ops.tape8_pack(meta(1, W, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="width"):
            ops.tape8_empty(1, W, device="meta")
        with pytest.raises(ValueError, match="columns"):
            ops.tape8_linear_bwd(meta(1, W), ops.tape8_empty(1, 40, device="meta"), meta(W, 40))
    nb = (wide + 31) // 32
    with pytest.raises(ValueError, match="width"):
        ops.tape8_unpack(ops.Tape8(meta(1, 32 * nb, dtype=torch.uint8), meta(1, nb, dtype=torch.uint8), wide))


def test_the_workspace_of_a_wide_weight():
    n = C.c_long(0)
    entry = _lib.lib().magnet_tape8_linear_bwd_workspace
    for M in (1, 100, 1 << 20):
        for K in (128, 4096, 4097, 200_000, 1 << 24, (1 << 31) - 256):
            assert entry(C.c_long(M), C.c_long(128), C.c_long(K), C.byref(n)) == 0
            assert 0 < 4 * n.value <= 512 << 20, (M, K, n.value)
    assert entry(C.c_long(1), C.c_long(1), C.c_long((1 << 31) - 1), C.byref(n)) == -2
    assert entry(C.c_long(1), C.c_long((1 << 31) - 1), C.c_long(1), C.byref(n)) == -2
