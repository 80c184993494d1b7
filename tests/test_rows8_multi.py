"""Rotated writes, chunk and shared-prefix attention and sinks of the 8-bit K/V row store without a GPU: refusals, which come
before any launch, and workspace queries; the oracle's rotation against closed forms."""
import numpy as np
import pytest

from fathom_amd import _lib
from oracle import rows8_oracle as R

FAR = 2 ** 63 - 1
K8, V8, KS, VS = 1 << 22, 1 << 23, 1 << 24, 1 << 25  # made-up addresses


def _refused(fn, args, status, text):
    L = _lib.lib()
    assert getattr(L, fn)(*args.values()) == status
    assert text in L.fathom_last_error(), L.fathom_last_error()


def _rotate(**kw):
    a = dict(q=1 << 20, K=1 << 21, V=1 << 21, dtype=_lib.DT_BF16, qr=128 * 8, qh=128, qt=128, kr=128 * 8, kt=128, vr=128 * 8, vt=128,
             pos=None, at=0, offset=None, shift=0, inv=1 << 19, turn=128, qw=None, kw=None, wdt=_lib.DT_F32, eps=1e-6, BH=2, G=4,
             T=8, D=128, cap=64, code=_lib.DT_E4M3, k8=K8, v8=V8, ks=KS, vs=VS, out=1 << 26, kout=None, stream=None)
    assert not set(kw) - set(a)
    return {**a, **kw}


@pytest.mark.parametrize("bad, text", [
    (dict(q=None), b"null"), (dict(V=None), b"null"), (dict(out=None), b"null"), (dict(inv=None), b"null"), (dict(ks=None), b"null"),
    (dict(dtype=7), b"dtype"), (dict(code=_lib.DT_F16), b"code_dtype"), (dict(qw=1 << 18, wdt=4), b"weight_dtype"),
    (dict(kw=1 << 18, wdt=-1), b"weight_dtype"), (dict(D=96), b"D=96"), (dict(BH=0), b"BH"), (dict(G=0), b"G=0"), (dict(G=65536), b"G="),
    (dict(T=-1), b"T=-1"), (dict(T=65), b"T=65"), (dict(T=2 ** 27 + 1, cap=2 ** 30), b"at most"), (dict(at=57), b"outside"),
    (dict(at=-1), b"outside"), (dict(at=FAR), b"outside"), (dict(shift=2 ** 31), b"offset"), (dict(shift=-FAR), b"offset"),
    (dict(turn=8), b"multiple of 16"), (dict(turn=144), b"multiple of 16"), (dict(turn=-16), b"multiple of 16"),
    (dict(D=64, turn=128), b"multiple of 16"), (dict(eps=-1e-6), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(eps=float("inf")), b"eps"), (dict(q=(1 << 20) + 8), b"16 bytes"), (dict(kout=(1 << 27) + 8), b"16 bytes"),
    (dict(qh=132), b"16 bytes"), (dict(vt=4), b"16 bytes"), (dict(k8=K8 + 4), b"aligned")])
def test_write_rotated_refusals(bad, text):
    _refused("fathom_rows8_write_rotated", _rotate(**bad), _lib.ERR_INVALID, text)


def test_write_rotated_of_no_token_is_no_launch():
    assert _lib.lib().fathom_rows8_write_rotated(*_rotate(T=0, q=None, K=None, V=None, out=None).values()) == _lib.OK


def _sink(**kw):
    a = dict(q=1 << 20, q_dtype=_lib.DT_F32, k8=K8, v8=V8, ks=KS, vs=VS, code=_lib.DT_I8, BH=2, G=4, D=128, cap=100000, lens=None,
             n=100000, window=50000, sinks=4, scale=0.1, softcap=0.0, slopes=None, out=1 << 26, ws=None, wsb=0, stream=None)
    assert not set(kw) - set(a)
    return {**a, **kw}


@pytest.mark.parametrize("bad, text, status", [
    (dict(q=None), b"null", _lib.ERR_INVALID), (dict(window=-1), b"window", _lib.ERR_INVALID), (dict(sinks=-1), b"sinks", _lib.ERR_INVALID),
    (dict(n=100001), b"length", _lib.ERR_INVALID), (dict(), b"workspace", _lib.ERR_WORKSPACE),
    (dict(sinks=FAR), b"workspace", _lib.ERR_WORKSPACE), (dict(window=FAR, sinks=FAR), b"workspace", _lib.ERR_WORKSPACE),
    (dict(ws=(1 << 28) + 8, wsb=1 << 34), b"aligned", _lib.ERR_INVALID)])
def test_sink_attention_refusals(bad, text, status):
    _refused("fathom_rows8_sink_attention", _sink(**bad), status, text)


def _chunk(**kw):
    a = dict(q=1 << 20, q_dtype=_lib.DT_BF16, qr=4 * 8 * 128, qh=8 * 128, qt=128, k8=K8, v8=V8, ks=KS, vs=VS, code=_lib.DT_E4M3, BH=2,
             G=4, T=8, D=128, cap=100000, lens=None, n=100000, window=0, sinks=0, scale=0.1, softcap=0.0, slopes=None, out=1 << 26,
             ws=None, wsb=0, stream=None)
    assert not set(kw) - set(a)
    return {**a, **kw}


@pytest.mark.parametrize("bad, text, status", [
    (dict(q=None), b"null", _lib.ERR_INVALID), (dict(out=None), b"null", _lib.ERR_INVALID), (dict(q_dtype=3), b"q_dtype", _lib.ERR_INVALID),
    (dict(k8=None), b"null", _lib.ERR_INVALID), (dict(D=32), b"D=32", _lib.ERR_INVALID), (dict(BH=65536), b"BH", _lib.ERR_INVALID),
    (dict(G=0), b"G=0", _lib.ERR_INVALID), (dict(T=-1), b"T=-1", _lib.ERR_INVALID), (dict(T=2 ** 20), b"queries", _lib.ERR_INVALID),
    (dict(T=FAR), b"queries", _lib.ERR_INVALID), (dict(n=-1), b"length", _lib.ERR_INVALID), (dict(n=100001), b"length", _lib.ERR_INVALID),
    (dict(window=-1), b"window", _lib.ERR_INVALID), (dict(sinks=-1), b"sinks", _lib.ERR_INVALID),
    (dict(softcap=-1.0), b"softcap", _lib.ERR_INVALID), (dict(softcap=float("nan")), b"softcap", _lib.ERR_INVALID),
    (dict(q=(1 << 20) + 2), b"aligned", _lib.ERR_INVALID), (dict(out=(1 << 26) + 2), b"16 bytes", _lib.ERR_INVALID),
    (dict(qt=4), b"16 bytes", _lib.ERR_INVALID), (dict(), b"workspace", _lib.ERR_WORKSPACE),
    (dict(ws=(1 << 28) + 8, wsb=1 << 34), b"aligned", _lib.ERR_INVALID)])
def test_chunk_attention_refusals(bad, text, status):
    _refused("fathom_rows8_chunk_attention", _chunk(**bad), status, text)


def test_chunk_attention_of_no_token_is_no_launch():
    assert _lib.lib().fathom_rows8_chunk_attention(*_chunk(T=0, q=None, out=None).values()) == _lib.OK


def _shared(**kw):
    a = dict(q=1 << 20, q_dtype=_lib.DT_F32, pk8=K8, pv8=V8, pks=KS, pvs=VS, pBH=2, pcap=10000, plens=None, pn=10000, k8=K8, v8=V8, ks=KS,
             vs=VS, code=_lib.DT_E4M3, seqs=3, G=4, D=128, cap=1000, lens=None, n=1000, scale=0.1, softcap=0.0, slopes=None,
             out=1 << 26, ws=1 << 28, wsb=1 << 34, stream=None)
    assert not set(kw) - set(a)
    return {**a, **kw}


@pytest.mark.parametrize("bad, text, status", [
    (dict(q=None), b"null", _lib.ERR_INVALID), (dict(pk8=None), b"null", _lib.ERR_INVALID), (dict(v8=None), b"null", _lib.ERR_INVALID),
    (dict(pBH=0), b"BH", _lib.ERR_INVALID), (dict(seqs=0), b"sequences", _lib.ERR_INVALID), (dict(seqs=32768), b"sequences", _lib.ERR_INVALID),
    (dict(seqs=FAR), b"sequences", _lib.ERR_INVALID), (dict(G=0), b"G=0", _lib.ERR_INVALID), (dict(seqs=32767, G=128), b"queries", _lib.ERR_INVALID),
    (dict(pn=10001), b"prefix length", _lib.ERR_INVALID), (dict(pn=-1), b"prefix length", _lib.ERR_INVALID),
    (dict(n=1001), b"length", _lib.ERR_INVALID), (dict(softcap=float("inf")), b"softcap", _lib.ERR_INVALID),
    (dict(ws=None), b"workspace", _lib.ERR_WORKSPACE), (dict(wsb=100), b"workspace", _lib.ERR_WORKSPACE),
    (dict(ws=(1 << 28) + 8), b"aligned", _lib.ERR_INVALID), (dict(q_dtype=4), b"q_dtype", _lib.ERR_INVALID)])
def test_shared_attention_refusals(bad, text, status):
    _refused("fathom_rows8_shared_attention", _shared(**bad), status, text)


def test_shared_workspace_is_checked_to_its_end():
    """One byte less than the query asks for the same lengths is refused: by the prefix's part or by the other one."""
    L = _lib.lib()
    need = L.fathom_rows8_shared_attention_workspace_bytes(2, 3, 4, 128, 10000, 1000)
    assert need > 0
    prefix = need - L.fathom_rows8_attention_workspace_bytes(6, 4, 128, 1000)
    for wsb in (0, 16, prefix // 2):
        _refused("fathom_rows8_shared_attention", _shared(wsb=wsb), _lib.ERR_WORKSPACE, b"workspace")


@pytest.mark.parametrize("G, T", [(1, 1), (4, 1), (4, 8), (4, 9), (7, 300), (12, 3001)])
@pytest.mark.parametrize("BH", [1, 7, 64, 300])
def test_workspace_sizes_do_not_fall_as_positions_grow(BH, G, T):
    """Callers ask for the next power of two and keep the answer."""
    L = _lib.lib()
    at = sorted({n + d for n in [1 << i for i in range(27)] + [300, 1088, 5000] for d in (-1, 0, 1) if n + d > 0})
    for D in (64, 128):
        sizes = [L.fathom_rows8_chunk_attention_workspace_bytes(BH, G, T, D, n) for n in at]
        assert sizes == sorted(sizes) and all(b % 16 == 0 for b in sizes)
        if BH * T > 65535:
            continue
        sizes = [[L.fathom_rows8_shared_attention_workspace_bytes(BH, T, G, D, n, m) for n in at] for m in at[::9]]
        assert all(row == sorted(row) for row in sizes) and all(list(c) == sorted(c) for c in zip(*sizes))


def test_workspace_queries_at_the_ends():
    L = _lib.lib()
    chunk, shared = L.fathom_rows8_chunk_attention_workspace_bytes, L.fathom_rows8_shared_attention_workspace_bytes
    most = 2 ** 31 - 65
    for BH, G, T, D in ((65536, 4, 1, 128), (4, 65536, 1, 128), (4, 4, 1, 96), (4, 4, 0, 128), (4, 4, FAR, 128), (4, 65535, 33, 128),
                        (2 ** 32, 2 ** 32, 1, 128), (-1, 4, 4, 128)):
        assert chunk(BH, G, T, D, 100000) == 0
    assert chunk(4, 4, 4, 128, FAR) == chunk(4, 4, 4, 128, most) > 0
    assert chunk(4, 4, 4, 128, 0) == chunk(4, 4, 4, 128, -FAR) == 0
    for H, B, G, D in ((65536, 1, 4, 128), (4, 20000, 4, 128), (4, 0, 4, 128), (4, FAR, 4, 128), (4, 4, 65536, 128), (4, 4, 4, 32)):
        assert shared(H, B, G, D, 1000, 1000) == 0
    assert shared(4, 4, 4, 128, FAR, FAR) == shared(4, 4, 4, 128, most, most) > 0
    assert shared(4, 4, 4, 128, -1, -1) == shared(4, 4, 4, 128, 0, 0) > 0


# ----------------------------------------------------------------------------- the oracle
def test_oracle_rotation_closed_forms():
    x = np.zeros((3, 16))
    x[:, 0], x[:, 15] = 1.0, 5.0
    got = R.rotated(x, np.array([2, 3, 4]), np.array([np.pi / 2] * 4), None)  # r = 8: channels 0 and 4; 15 stays
    assert np.allclose(got[:, 0], [-1, 0, 1]) and np.allclose(got[:, 4], [0, -1, 0]) and np.allclose(got[:, 15], 5)
    got = R.rotated(np.full((1, 4), 3.0), np.array([7]), np.zeros(0), np.array([1.0, 2.0, 0.0, -1.0]))
    assert np.allclose(got, [[1, 2, 0, -1]])


@pytest.mark.parametrize("entry", ["chunk", "shared"])
@pytest.mark.parametrize("BH, G, T", [(1, 4, 64), (6, 8, 300), (1, 4, 9), (2, 8, 1024), (4, 7, 33), (64, 4, 128)])
def test_a_workspace_serves_every_kind_of_call(entry, BH, G, T):
    """Queries of each type, with a cap, a bias or neither, take what the query's size holds; a fourth of it is refused to some.
    (The workspace is 8 bytes off, so that no call gets to its launch.)"""
    n = 65536
    L = _lib.lib()
    if entry == "chunk":
        need = L.fathom_rows8_chunk_attention_workspace_bytes(BH, G, T, 128, n)
        args = _chunk(BH=BH, G=G, T=T, cap=n, n=0, lens=1 << 29)
    else:
        need = L.fathom_rows8_shared_attention_workspace_bytes(BH, T, G, 128, n, 0)
        args = _shared(pBH=BH, seqs=T, G=G, pcap=n, pn=0, plens=1 << 29, n=0)
    refused = 0
    for q_dtype in (_lib.DT_F32, _lib.DT_F16, _lib.DT_BF16):
        for softcap, slopes in ((0.0, None), (30.0, None), (0.0, 1 << 29), (1e30, None)):
            call = {**args, "q_dtype": q_dtype, "softcap": softcap, "slopes": slopes, "ws": (1 << 28) + 8}
            _refused(f"fathom_rows8_{entry}_attention", {**call, "wsb": need}, _lib.ERR_INVALID, b"aligned")
            refused += getattr(L, f"fathom_rows8_{entry}_attention")(*{**call, "wsb": need // 4}.values()) == _lib.ERR_WORKSPACE
    assert refused


@pytest.mark.parametrize("entry", ["chunk", "shared"])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_scales_that_are_not_finite_are_refused(entry, scale):
    args = _chunk(scale=scale) if entry == "chunk" else _shared(scale=scale)
    _refused(f"fathom_rows8_{entry}_attention", args, _lib.ERR_INVALID, b"scale")


@pytest.mark.parametrize("lens", [None, 1 << 29])
def test_the_shared_workspace_holds_the_rows_own_part_too(lens):
    """Sizes from what the prefix's part takes up to one byte less than both take are refused by the check of the rows' own part, before
    any launch; what the query answers holds both.  (The least size that the prefix's part takes is found with an address that is 8
    bytes off, which is refused behind that check.)"""
    L = _lib.lib()
    args = _shared(cap=100000, n=100000, lens=lens)

    def status(wsb, ws=1 << 28):
        return L.fathom_rows8_shared_attention(*{**args, "ws": ws, "wsb": wsb}.values())

    need = L.fathom_rows8_shared_attention_workspace_bytes(2, 3, 4, 128, 10000, 100000)
    low, high = 0, need  # refused for its size, and not
    while high - low > 1:
        mid = (low + high) // 2
        low, high = (mid, high) if status(mid, (1 << 28) + 8) == _lib.ERR_WORKSPACE else (low, mid)
    assert status(high) == _lib.ERR_WORKSPACE
    message = L.fathom_last_error()
    assert b"more than" not in message and b"workspace 0 bytes" in message
    own = int(message.split()[-1])
    assert own > 0 and need >= high + own
    for wsb in (high + 1, high + own // 2, high + own - 1):
        _refused("fathom_rows8_shared_attention", {**args, "wsb": wsb}, _lib.ERR_WORKSPACE, b"workspace %d bytes, need %d" % (wsb - high, own))
