"""The 8-bit K/V row store without a GPU: its oracle's code formats against torch's, the
oracle's growth of scales, and refusals."""
import numpy as np
import pytest
import torch

from fathom_amd import _lib
from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R


def test_oracle_e4m3_codes_equal_torch():
    b = torch.arange(256, dtype=torch.uint8)
    v = b.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.decode(b.numpy(), "e4m3"), v, equal_nan=True)
    g = torch.Generator().manual_seed(0)
    y = torch.cat([torch.randn(20000, generator=g) * s for s in (1e-3, 1.0, 100.0)]).clamp(-448, 448)
    t = torch.from_numpy(v[:127])
    mid = ((t[1:] + t[:-1]) / 2).float()  # ties
    y = torch.cat([y, t.float(), mid, -mid, torch.tensor([0.0, -0.0])])
    assert np.array_equal(R.encode(y.numpy(), "e4m3"), y.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert R.encode(np.array([np.nan, np.inf, -np.inf]), "e4m3").tolist() == [0x7F, 0x7E, 0xFE]


def test_oracle_int8_codes():
    y = np.array([0.5, 1.5, -0.5, -2.5, 127.4, 500.0, -500.0, np.nan, np.inf])
    assert R.decode(R.encode(y, "int8"), "int8").tolist() == [0, 2, 0, -2, 127, 127, -127, 0, 127]


def test_oracle_scale_growth():
    assert R.grown(np.float32(0.75), np.float32(0.75)) == (np.float32(0.75), 0)
    assert R.grown(np.float32(0.75), np.float32(0.76)) == (np.float32(1.5), 1)
    assert R.grown(np.float32(0.75), np.float32(1.5)) == (np.float32(1.5), 1)
    assert R.grown(np.float32(0.75), np.float32(5.0)) == (np.float32(6.0), 3)


def test_oracle_attention_closed_forms():
    rng = np.random.default_rng(0)
    K, V, q = rng.standard_normal((9, 64)), rng.standard_normal((9, 64)), rng.standard_normal(64)
    out, _ = R.attention(q, K, V, [4], 9, 0.125)
    assert np.allclose(out, V[4])
    out, _ = R.attention(0 * q, K, V, [1, 2, 2], 9, 0.125)
    assert np.allclose(out, (V[1] + 2 * V[2]) / 3)
    out, _ = R.attention(0 * q, K, V, [7, 8], 9, 0.125, slope=np.log(3.0))  # one token further back: a third
    assert np.allclose(out, (V[7] + 3 * V[8]) / 4)
    out, _ = R.attention(q * 1e6, K, V, list(range(9)), 9, 0.125, softcap=1e-9)  # every score at the cap: +-1e-9
    assert np.allclose(out, V.mean(0))


def test_host_tensors_are_refused():
    z = torch.zeros(2, 64, 128, dtype=torch.int8)
    with pytest.raises(ValueError, match="GPU"):
        RowStore8(z, z, torch.zeros(2, 1), torch.zeros(2, 1))


def _write_args(**kw):
    """Arguments of fathom_rows8_write over made-up addresses, for calls that are refused before any launch."""
    a = dict(K=1 << 20, V=1 << 21, dtype=_lib.DT_BF16, krs=128 * 8, kts=128, vrs=128 * 8, vts=128, pos=None, at=0, BH=2, T=8,
             D=128, cap=64, code=_lib.DT_E4M3, k8=1 << 22, v8=1 << 23, ks=1 << 24, vs=1 << 25, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad, text", [
    (dict(K=None), b"null"), (dict(k8=None), b"null"), (dict(dtype=7), b"dtype"), (dict(code=_lib.DT_F16), b"code_dtype"),
    (dict(D=96), b"D=96"), (dict(BH=0), b"BH"), (dict(BH=65536), b"BH"), (dict(cap=0), b"cap"), (dict(T=65), b"T=65"),
    (dict(T=-1), b"T=-1"), (dict(at=57), b"outside"), (dict(at=-1), b"outside"), (dict(K=(1 << 20) + 8), b"16 bytes"),
    (dict(kts=132), b"16 bytes"), (dict(k8=(1 << 22) + 4), b"aligned"), (dict(ks=(1 << 24) + 2), b"aligned")])
def test_write_refusals(bad, text):
    L = _lib.lib()
    assert L.fathom_rows8_write(*_write_args(**bad)) == _lib.ERR_INVALID
    assert text in L.fathom_last_error()


def test_write_of_no_token_is_no_launch():
    assert _lib.lib().fathom_rows8_write(*_write_args(T=0, K=None, V=None)) == _lib.OK


def _read_args(**kw):
    a = dict(k8=1 << 22, v8=1 << 23, ks=1 << 24, vs=1 << 25, code=_lib.DT_I8, BH=2, cap=64, D=64, idx=None, pos=None, at=0, R=8,
             dtype=_lib.DT_F32, K=1 << 20, V=1 << 21, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad, text", [
    (dict(v8=None), b"null"), (dict(V=None), b"null"), (dict(dtype=3), b"dtype"), (dict(R=-1), b"rows"), (dict(R=1 << 31), b"rows"),
    (dict(K=(1 << 20) + 4), b"aligned"), (dict(code=9), b"code_dtype")])
def test_read_refusals(bad, text):
    L = _lib.lib()
    assert L.fathom_rows8_read(*_read_args(**bad)) == _lib.ERR_INVALID
    assert text in L.fathom_last_error()


def _attn_args(**kw):
    a = dict(q=1 << 20, q_dtype=_lib.DT_F32, k8=1 << 22, v8=1 << 23, ks=1 << 24, vs=1 << 25, code=_lib.DT_I8, BH=2, G=4, D=128,
             cap=100000, lens=None, n=100000, window=0, scale=0.1, softcap=0.0, slopes=None, out=1 << 26, ws=None, wsb=0,
             stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad, text, status", [
    (dict(q=None), b"null", _lib.ERR_INVALID), (dict(out=None), b"null", _lib.ERR_INVALID),
    (dict(q_dtype=5), b"q_dtype", _lib.ERR_INVALID), (dict(G=0), b"G=0", _lib.ERR_INVALID),
    (dict(G=65536), b"G=", _lib.ERR_INVALID), (dict(n=100001), b"length", _lib.ERR_INVALID),
    (dict(n=-1), b"length", _lib.ERR_INVALID), (dict(window=-1), b"window", _lib.ERR_INVALID),
    (dict(softcap=-1.0), b"softcap", _lib.ERR_INVALID), (dict(softcap=float("nan")), b"softcap", _lib.ERR_INVALID),
    (dict(softcap=float("inf")), b"softcap", _lib.ERR_INVALID),
    (dict(q=(1 << 20) + 4), b"aligned", _lib.ERR_INVALID), (dict(D=32), b"D=32", _lib.ERR_INVALID),
    (dict(ws=(1 << 28) + 8, wsb=1 << 34), b"aligned", _lib.ERR_INVALID), (dict(), b"workspace", _lib.ERR_WORKSPACE)])
def test_attention_refusals(bad, text, status):
    L = _lib.lib()
    assert L.fathom_rows8_attention(*_attn_args(**bad)) == status
    assert text in L.fathom_last_error()


@pytest.mark.parametrize("bad, text, status", [
    (dict(idx=None), b"null", _lib.ERR_INVALID), (dict(k=-1), b"k=-1", _lib.ERR_INVALID),
    (dict(k=1 << 30), b"k=", _lib.ERR_INVALID), (dict(k=1 << 20), b"workspace", _lib.ERR_WORKSPACE),
    (dict(k=1 << 20, ws=(1 << 28) + 4, wsb=1 << 34), b"aligned", _lib.ERR_INVALID)])
def test_gather_attention_refusals(bad, text, status):
    a = dict(q=1 << 20, q_dtype=_lib.DT_F32, idx=1 << 27, k8=1 << 22, v8=1 << 23, ks=1 << 24, vs=1 << 25, code=_lib.DT_I8, BH=2,
             G=4, k=512, D=128, cap=1000, lens=None, n=1000, scale=0.1, softcap=0.0, slopes=None, out=1 << 26, ws=None, wsb=0,
             stream=None)
    a.update(bad)
    L = _lib.lib()
    assert L.fathom_rows8_gather_attention(*a.values()) == status
    assert text in L.fathom_last_error()


def test_workspace_queries():
    L = _lib.lib()
    assert L.fathom_rows8_attention_workspace_bytes(0, 4, 128, 1000) == 0
    assert L.fathom_rows8_attention_workspace_bytes(1, 1, 128, 0) == 0
    assert L.fathom_rows8_attention_workspace_bytes(8, 4, 128, 1 << 20) > 0
    assert L.fathom_rows8_gather_attention_workspace_bytes(1, 1, 128, 1) == 0


@pytest.mark.parametrize("G", [1, 8, 9, 40])
@pytest.mark.parametrize("BH", [1, 7, 64, 300, 5000])
def test_workspace_sizes_do_not_fall_as_positions_grow(BH, G):
    """Callers ask for the next power of two and keep the answer."""
    L = _lib.lib()
    at = sorted({n + d for n in [1 << i for i in range(27)] + [300, 1088, 1089, 5000] for d in (-1, 0, 1) if n + d > 0})
    for query in (L.fathom_rows8_attention_workspace_bytes, L.fathom_rows8_gather_attention_workspace_bytes):
        sizes = [query(BH, G, 128, n) for n in at]
        assert sizes == sorted(sizes) and all(b % 4 == 0 for b in sizes)
