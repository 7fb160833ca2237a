"""Refusals of the seam's backward entry point that take branch and residual: each returns before any CUDA call."""
import pytest

import __graft_entry__ as entry
from dcnv4_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.lib()


def _bwd(lib, gy=0x1000, gh=None, x=0x2000, res=0x2800, mean=0x3000, rstd=0x4000, w=0x5000, s=None, gr=0x7000, gx=None,
         gw=0x8000, gb=0x9000, ws=0xa000, ws_bytes=1 << 30, dtype=2, param=0, rows=4, C=16, per=4):
    return lib.dcnv4b200_add_layernorm_bwd(gy, gh, x, res, mean, rstd, w, s, gr, gx, gw, gb, ws, ws_bytes, dtype, param, rows,
                                           C, per, None)


def test_refuses(lib):
    assert _bwd(lib, dtype=0) == -2 and _bwd(lib, dtype=3) == -2 and _bwd(lib, dtype=1, param=2) == -2
    assert _bwd(lib, rows=-1) == -3 and _bwd(lib, C=0) == -3 and _bwd(lib, s=0x100, per=3) == -3
    assert _bwd(lib, C=8193) == -6 and _bwd(lib, rows=(1 << 30) + 1) == -9
    for name in ("gy", "x", "res", "mean", "rstd", "w", "gr", "gw", "gb"):
        assert _bwd(lib, **{name: None}) == -1, name
    assert _bwd(lib, s=0x100) == -1                       # a scaled branch without room for its gradient
    for name in ("gy", "gh", "x", "res", "gr", "gx"):
        assert _bwd(lib, **{name: 0x7001}) == -4, name
    assert _bwd(lib, ws=None) == -5 and _bwd(lib, ws_bytes=16) == -5 and _bwd(lib, ws=0xa008) == -4
