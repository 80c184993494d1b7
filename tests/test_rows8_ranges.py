"""The row store's C entry points at the ends of their integer ranges, without a GPU: refusals come before any launch."""
import pytest

from fathom_amd import _lib
from test_rows8 import _attn_args, _read_args, _write_args

FAR = 2 ** 63 - 1


@pytest.mark.parametrize("at, T", [(FAR, 8), (FAR - 7, 8), (FAR, 1), (FAR - 64, 64), (-FAR - 1, 8), (57, 8)])
def test_write_places_do_not_wrap(at, T):
    L = _lib.lib()
    assert L.fathom_rows8_write(*_write_args(at=at, T=T)) == _lib.ERR_INVALID
    assert b"outside" in L.fathom_last_error()
