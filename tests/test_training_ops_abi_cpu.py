"""Refusals of the training-step entry points: every bad argument returns before any CUDA call (the pointers below are
never dereferenced), so this runs without a GPU."""
import pytest

import __graft_entry__ as entry
from dcnv4_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.lib()


def _fwd(lib, x=0x1000, res=0x2000, w=0x3000, b=0x4000, gamma=0x5000, s=None, y=0x6000, h=0x7000, mean=0x8000,
         rstd=0x9000, mode=0, dtype=0, out=0, param=0, rows=4, C=16, per=4, act=0):
    return lib.dcnv4b200_layernorm_train_fwd(x, res, w, b, gamma, s, y, h, mean, rstd, mode, dtype, out, param, rows, C,
                                             per, 1e-6, act, None)


def _bwd(lib, gy=0x1000, gh=None, x=0x2000, mean=0x3000, rstd=0x4000, w=0x5000, b=0x6000, gamma=None, s=None, gx=0x7000,
         branch=None, gw=0x8000, gb=0x9000, gs=None, ws=0xa000, ws_bytes=1 << 30, mode=0, dtype=0, out=0, param=0, rows=4,
         C=16, per=4, act=0):
    return lib.dcnv4b200_layernorm_train_bwd(gy, gh, x, mean, rstd, w, b, gamma, s, gx, branch, gw, gb, gs, ws, ws_bytes,
                                             mode, dtype, out, param, rows, C, per, act, None)


def test_layernorm_forward_refuses(lib):
    assert _fwd(lib, mode=3) == -6 and _fwd(lib, mode=-1) == -6
    assert _fwd(lib, act=1, mode=1) == -6 and _fwd(lib, act=2) == -6
    assert _fwd(lib, dtype=3) == -2
    assert _fwd(lib, dtype=0, out=1) == -2                # fp32 in, fp16 out
    assert _fwd(lib, dtype=1, out=2) == -2
    assert _fwd(lib, dtype=1, out=0, param=2) == -2
    assert _fwd(lib, rows=-1) == -3 and _fwd(lib, C=0) == -3
    assert _fwd(lib, C=8193) == -6
    assert _fwd(lib, rows=1 << 31) == -9
    assert _fwd(lib, mode=1, s=0x100, per=0) == -3 and _fwd(lib, mode=1, s=0x100, per=3) == -3
    assert _fwd(lib, x=None) == -1 and _fwd(lib, mean=None) == -1 and _fwd(lib, w=None) == -1
    assert _fwd(lib, mode=1, res=None) == -1 and _fwd(lib, mode=2, h=None) == -1
    assert _fwd(lib, x=0x1002) == -4 and _fwd(lib, w=0x3001) == -4 and _fwd(lib, s=0x102) == -4
    assert _fwd(lib, rows=0) == 0


def test_layernorm_row_limit(lib):
    """Row numbers plus a stride of the grid stay within 32 bits."""
    most = 1 << 30
    assert _fwd(lib, rows=most + 1) == -9 and _bwd(lib, rows=most + 1) == -9
    need = lib.dcnv4b200_layernorm_train_bwd_workspace_bytes
    assert need(0, most, 1) > 0 and need(0, most + 1, 1) == 0


def test_layernorm_backward_refuses(lib):
    assert _bwd(lib, gx=None) == -1 and _bwd(lib, gw=None) == -1 and _bwd(lib, gy=None) == -1
    assert _bwd(lib, mode=1, gamma=0x100) == -1           # layer scale without room for its gradient
    assert _bwd(lib, mode=2, s=0x100) == -1               # scaled branch without room for its gradient
    assert _bwd(lib, mode=2, dtype=1, out=0) == -1        # likewise where the types differ
    assert _bwd(lib, ws=None) == -5 and _bwd(lib, ws_bytes=16) == -5
    assert _bwd(lib, ws=0xa008) == -4 and _bwd(lib, gx=0x7002) == -4
    assert _bwd(lib, C=9000) == -6 and _bwd(lib, act=1, mode=2) == -6


def test_layernorm_workspace(lib):
    need = lib.dcnv4b200_layernorm_train_bwd_workspace_bytes
    assert need(0, 0, 64) == 0 and need(7, 4, 64) == 0 and need(0, 4, 9000) == 0
    for dtype in (0, 1, 2):
        assert 2 * 64 * 4 <= need(dtype, 1, 64) <= need(dtype, 100000, 64)
    assert need(0, 2 ** 31 - 1, 8192) < 64 << 20


def test_functions_refuse_cpu_tensors():
    import torch
    from dcnv4_b200 import ops
    x, w = torch.zeros(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layer_norm_train_forward(x, w, w, 1e-6)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layer_norm_residual_forward(x, x, w, w, 1e-6)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.add_layer_norm_forward(x, x, w, w, 1e-6)


def _ns(lib, x=0x1000, out=0x2000, ws=0x4000, ws_bytes=1 << 40, dtype=0, batch=1, m=300, n=200, steps=5):
    return lib.dcnv4b200_newton_schulz(x, out, ws, ws_bytes, dtype, batch, m, n, steps, 3.4445, -4.775, 2.0315, 1e-7, None)


def test_newton_schulz_refuses(lib):
    assert _ns(lib, dtype=3) == -2
    assert _ns(lib, batch=-1) == -3 and _ns(lib, m=0) == -3 and _ns(lib, n=0) == -3 and _ns(lib, steps=0) == -3
    assert _ns(lib, m=65537) == -6 and _ns(lib, batch=65536) == -6 and _ns(lib, steps=101) == -6
    assert _ns(lib, batch=0) == 0
    assert _ns(lib, x=None) == -1 and _ns(lib, out=None) == -1
    assert _ns(lib, x=0x1002) == -4 and _ns(lib, out=0x2001) == -4 and _ns(lib, ws=0x4008) == -4
    assert _ns(lib, ws=None) == -5 and _ns(lib, ws_bytes=1000) == -5


def test_newton_schulz_workspace(lib):
    need = lib.dcnv4b200_newton_schulz_workspace_bytes
    assert need(0, 64, 64) == 0 and need(1, 0, 64) == 0 and need(1, 64, 70000) == 0
    assert need(3, 65, 257) >= 3 * (4 * 65 * 264 + 2 * 65 * 72) * 2
    assert need(3, 128, 256) == 0 and need(9, 256, 128) == 0    # held by one block each
    assert need(65535, 65536, 65536) > 1 << 47             # no 32-bit overflow


def test_newton_schulz_refuses_cpu_tensors():
    import torch
    from dcnv4_b200 import ops
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.newton_schulz(torch.zeros(3, 8))
