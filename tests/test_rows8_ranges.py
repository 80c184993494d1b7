"""The row store's C entry points at the ends of their integer ranges, without a GPU: refusals come before any launch."""
import os
import subprocess
import sys

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


def test_workspace_queries_at_the_ends():
    """Shapes that the calls refuse need no workspace; positions and k past every store need what the longest do."""
    L = _lib.lib()
    for query, most in ((L.fathom_rows8_attention_workspace_bytes, 2 ** 31 - 65),
                        (L.fathom_rows8_gather_attention_workspace_bytes, (2 ** 31 - 1) // 4)):
        for BH, G, D in ((65536, 4, 128), (4, 65536, 128), (4, 4, 96), (2 ** 32, 4, 128), (4, 2 ** 62, 128), (4, 4, 2 ** 62)):
            assert query(BH, G, D, 100000) == 0
        assert query(4, 4, 128, most) > 0
        assert query(4, 4, 128, FAR) == query(4, 4, 128, 2 ** 40) == query(4, 4, 128, most)
        assert query(2, 4, 128, -5) == query(2, -4, 128, 5) == 0


def test_workspace_queries_do_not_divide_by_zero():
    """2^32 x 2^32 heads, whose product is 0 in 64 bits: asked in a process of its own, as a division by it ends one."""
    code = ("from fathom_amd import _lib; L = _lib.lib(); "
            "print([q(2 ** 32, 2 ** 36, 128, 10 ** 6) for q in (L.fathom_rows8_attention_workspace_bytes, "
            "L.fathom_rows8_gather_attention_workspace_bytes)])")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "[0, 0]", (run.returncode, run.stderr[-500:])


@pytest.mark.parametrize("T", [2 ** 30 - 127, 2 ** 30, 2 ** 31 - 65])
def test_writes_longer_than_a_grid_are_refused(T):
    L = _lib.lib()
    assert L.fathom_rows8_write(*_write_args(T=T, cap=2 ** 31 - 65)) == _lib.ERR_INVALID
    assert f"T={T}".encode() in L.fathom_last_error()
