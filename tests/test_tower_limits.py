"""Pointers that the tower's C entry points cannot take, refused before any device work."""

import silvertorch_amd.ops._load_ops  # noqa: F401
from silvertorch_amd import capi


def test_int8_matmul_refuses_an_unaligned_workspace():
    """Codes are made in it with 8-byte stores and read in 16-byte pieces."""
    L = capi.lib()
    call = lambda ws: L.st_int8_matmul(16, 16, 4, 32, 16, 0, None, 5, 20, 20, None, 16, 0, ws, None)  # noqa: E731
    assert L.st_int8_matmul_workspace_bytes(0, 5, 4, 32) > 0
    for workspace in (1, 4, 8, 24):
        assert call(workspace) != 0
        assert "the workspace must be 16-byte aligned" in L.st_last_error().decode()
    assert call(None) != 0 and "null device pointer" in L.st_last_error().decode()
