"""What the tower's entry points cannot take, refused before any device work: pointers, types that do not agree."""

import pytest
import torch

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


def test_layer_norm_backward_refuses_a_weight_of_another_type():
    """The kernel would read it as weight_type."""
    h, stats = torch.zeros((3, 10)), torch.zeros((3, 3))
    for weight, weight_type in ((torch.ones(10).half(), torch.float32), (torch.ones(10), torch.bfloat16)):
        with pytest.raises(RuntimeError, match="weight must be of weight_type"):
            torch.ops.st.layer_norm_backward(h, None, h, weight, stats, None, 0.0, torch.float32, weight_type, [True] * 4)
