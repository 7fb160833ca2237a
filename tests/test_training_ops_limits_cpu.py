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


def test_sizes_beyond_32_bits_are_refused(lib, monkeypatch):
    """A C int would wrap: (1, 2^32 + 8) must not be taken for (1, 8).  The tensors here have one element of memory; the
    checks are those that a CUDA tensor meets."""
    monkeypatch.setattr(ops, "_check_tensor", lambda t, name: None)
    n = 2 ** 32 + 8
    wide = torch.zeros(1).expand(1, n)
    for x in (wide, wide.t(), torch.zeros(1).expand(65537, 4)):
        with pytest.raises(ValueError):
            ops.newton_schulz(x)
    with pytest.raises(ValueError):
        ops.newton_schulz(torch.zeros(4, 4), 2 ** 32 + 5)
    with pytest.raises(ValueError):
        ops.layer_norm_train_forward(wide, wide[0], wide[0], 1e-6)
    with pytest.raises(ValueError):
        ops.layer_norm_backward(wide, wide, torch.zeros(1), torch.ones(1), wide[0], wide[0])
