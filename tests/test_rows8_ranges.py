"""The row store's C entry points at the ends of their integer ranges, without a GPU: refusals come before any launch."""
import pytest

from fathom_amd import _lib
from test_rows8 import _write_args

FAR = 2 ** 63 - 1


@pytest.mark.parametrize("at, T", [(FAR, 8), (FAR - 7, 8), (FAR, 1), (FAR - 64, 64), (-FAR - 1, 8), (57, 8)])
def test_write_places_do_not_wrap(at, T):
    L = _lib.lib()
    assert L.fathom_rows8_write(*_write_args(at=at, T=T)) == _lib.ERR_INVALID
    assert b"outside" in L.fathom_last_error()


@pytest.mark.parametrize("G, k", [(4, 2 ** 62), (65535, FAR), (2, FAR), (4, 2 ** 29), (1, 2 ** 31)])
def test_selections_do_not_wrap(G, k):
    a = dict(q=1 << 20, q_dtype=_lib.DT_F32, idx=1 << 27, k8=1 << 22, v8=1 << 23, ks=1 << 24, vs=1 << 25, code=_lib.DT_I8, BH=2,
             G=G, k=k, D=128, cap=1000, lens=None, n=1000, scale=0.1, softcap=0.0, slopes=None, out=1 << 26, ws=1 << 28,
             wsb=1 << 50, stream=None)
    L = _lib.lib()
    assert L.fathom_rows8_gather_attention(*a.values()) == _lib.ERR_INVALID
    assert f"k={k}".encode() in L.fathom_last_error()
