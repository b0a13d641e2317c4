"""Limits of the retrieval head's arguments that are checked before any device work."""

import pytest
import torch

import silvertorch_amd.ops._load_ops  # noqa: F401

st = torch.ops.st


@pytest.mark.parametrize("group_size", [64, 1 << 40, (1 << 63) - 32])
def test_group_sizes_past_the_columns_make_one_group(group_size):
    packed, x = torch.zeros((5, 32), dtype=torch.uint8), torch.ones((3, 40))
    with pytest.raises(RuntimeError, match=r"scales must be \[5, 1\], got \[5, 2\]"):
        st.int4_matvec(packed, torch.ones((5, 2)), x, group_size)
