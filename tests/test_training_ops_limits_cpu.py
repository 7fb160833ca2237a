"""Limits of the training-step operators, without a GPU."""
import pytest
import torch

import __graft_entry__ as entry
from dcnv4_b200 import _lib, ops


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.lib()


def test_layernorm_workspace_at_the_largest_sizes(lib):
    """One (2, C) block per CTA, however many rows there are."""
    need = lib.dcnv4b200_layernorm_train_bwd_workspace_bytes
    for dtype in (0, 1, 2):
        assert 0 < need(dtype, 1 << 30, 8192) < 64 << 20
        assert need(dtype, (1 << 30) + 1, 8192) == 0
