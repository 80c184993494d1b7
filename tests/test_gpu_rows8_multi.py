"""Chunk attention, shared prefixes and windows with sinks over the 8-bit K/V row store on the GPU, against the oracle in
float64 within its bound of the kernels' arithmetic."""
import numpy as np
import pytest
import torch

from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R
from test_gpu_rows8 import BLK, CODES, DEV, _f32, _from_numpy, _rand

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of each type
# half a step below each type's smallest normal number, where steps no longer shrink with the value: float16's are 2^-24
FLOOR = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
BITS = {torch.float32: 22, torch.float16: 11, torch.bfloat16: 11}  # of a chunk's weights
PARTS = {torch.float32: 3, torch.float16: 1, torch.bfloat16: 1}


def _filled(BH, cap, D, code, seed=0, garbage_behind=None):
    """A store whose blocks were written at once, its numpy copy; bytes and scales behind `garbage_behind` [BH] are of any kind."""
    o = {"k8": np.zeros((BH, cap, D), np.uint8), "v8": np.zeros((BH, cap, D), np.uint8)}
    o["ks"], o["vs"] = np.zeros((2, BH, -(-cap // BLK)), np.float32)
    R.write(o, _f32(_rand((BH, cap, D), seed + 1)), _f32(_rand((BH, cap, D), seed + 2)), 0, code)
    if garbage_behind is not None:
        rng = np.random.default_rng(seed + 3)
        for b, n in enumerate(garbage_behind):
            for c in ("k8", "v8"):
                o[c][b, n:] = rng.integers(0, 256, (cap - n, D), dtype=np.uint8)
            for s in ("ks", "vs"):
                o[s][b, -(-n // BLK):] = np.nan
    return _from_numpy(o, code), o


def _values(o, code):
    return R.values(o["k8"], o["ks"], code), R.values(o["v8"], o["vs"], code)


def _check_chunk(got, q, o, code, lens, window=0, sinks=0, scale=None, softcap=0.0, slopes=None, every=1):
    """got [BH, G, T, d] against the oracle, every `every`-th token."""
    BH, G, T, D = got.shape
    K, V = _values(o, code)
    scale = D ** -0.5 if scale is None else scale
    got, half = got.double().cpu().numpy(), HALF[q.dtype]
    qf = q.double().cpu().numpy()
    for b in range(BH):
        n = int(lens[b])
        for i in range(0, T, every):
            p = n - T + i
            toks = R.sees(p, n, window, sinks)
            for g in range(G):
                ref, tol = R.many_attention(qf[b, g, i], K[b], V[b], toks, p + 1, scale, softcap,
                                            None if slopes is None else float(slopes[b, g]), BITS[q.dtype], PARTS[q.dtype])
                off = np.abs(got[b, g, i] - ref) - (tol + np.maximum((np.abs(ref) + tol) * half, FLOOR[q.dtype]))
                assert (off <= 0).all(), f"row {b} head {g} token {i} (place {p} of {n}): {off.max():.3g} over {tol.max():.3g}"


# ----------------------------------------------------------------------------- chunks
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G, T, lens", [(1, 1, [1, 64, 65]), (4, 8, [8, 0, 200]), (3, 43, [300, 43, 42]), (5, 131, [131, 333, 60])])
def test_chunk(code, dtype, D, G, T, lens):
    """One wave's tiles and four waves', whole and ragged, rows shorter than the chunk and empty ones."""
    st, o = _filled(3, 333, D, code, garbage_behind=lens)
    q = _rand((3 * G, T, D), 5, dtype).view(3, G, T, D)
    got = st.chunk_attention(q.to(DEV), torch.tensor(lens, device=DEV))
    assert got.dtype == dtype and got.shape == q.shape
    _check_chunk(got, q, o, code, lens, every=3 if T > 20 else 1)


@pytest.mark.parametrize("code, dtype, D", [("e4m3", torch.bfloat16, 128), ("int8", torch.float16, 64), ("e4m3", torch.float32, 64),
                                            ("int8", torch.float32, 128)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (64, 4), (63, 64), (100, 65), (130, 200), (500, 3), (10 ** 9, 7), (7, 10 ** 9)])
def test_chunk_windows_and_sinks(code, dtype, D, window, sinks):
    G, T, n = 4, 70, 400
    st, o = _filled(2, n, D, code, seed=3)
    q = _rand((2 * G, T, D), 6, dtype).view(2, G, T, D)
    got = st.chunk_attention(q.to(DEV), n, window=window, sinks=sinks)
    _check_chunk(got, q, o, code, [n, n], window, sinks, every=5)
    lens = [250, 90]
    got = st.chunk_attention(q.to(DEV), torch.tensor(lens, device=DEV), window=window, sinks=sinks)
    _check_chunk(got, q, o, code, lens, window, sinks, every=7)


@pytest.mark.parametrize("code, dtype, D", [("e4m3", torch.bfloat16, 128), ("int8", torch.float32, 64)])
@pytest.mark.parametrize("softcap, slopes, scale", [(30.0, False, None), (0.0, True, None), (5.0, True, 0.3), (2.0, False, -0.2),
                                                    (0.0, False, 0.0), (0.0, True, -0.1), (1e-25, False, None), (1e29, False, None)])
def test_chunk_caps_and_slopes(code, dtype, D, softcap, slopes, scale):
    G, T, n = 3, 50, 300
    st, o = _filled(2, n, D, code, seed=9)
    q = _rand((2 * G, T, D), 7, dtype).view(2, G, T, D)
    sl = 2.0 ** -torch.arange(1.0, 2 * G + 1).view(2, G) if slopes else None
    got = st.chunk_attention(q.to(DEV), n, scale=scale, softcap=softcap, slopes=None if sl is None else sl.to(DEV))
    cap = softcap if softcap < 1e27 else 0.0
    _check_chunk(got, q, o, code, [n, n], scale=scale, softcap=max(cap, 2.0 ** -64) if cap else 0.0, slopes=sl, every=4)
    if sl is not None:
        for shaped in (sl[0], sl[:, :1].double()):  # [G]; a view that expands
            one = st.chunk_attention(q.to(DEV), n, scale=scale, softcap=softcap, slopes=shaped.to(DEV))
            _check_chunk(one, q, o, code, [n, n], scale=scale, softcap=softcap, slopes=shaped.expand(2, G), every=25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("BH, G, T, n", [(1, 1, 1, 40000), (2, 4, 3, 20011), (1, 7, 40, 9000), (3, 2, 8, 4097)])
def test_chunk_in_splits(dtype, BH, G, T, n):
    """Few queries over long rows: the row is shared out over workgroups and joined."""
    st, o = _filled(BH, n, 128, "e4m3", seed=11)
    q = _rand((BH * G, T, 128), 8, dtype).view(BH, G, T, 128)
    _check_chunk(st.chunk_attention(q.to(DEV), n), q, o, "e4m3", [n] * BH, every=9)
    lens = [n - 5000 * b if b else 70 for b in range(BH)]
    got = st.chunk_attention(q.to(DEV), torch.tensor(lens, device=DEV))
    _check_chunk(got, q, o, "e4m3", lens, every=9)
    lens = [0] * BH
    assert not st.chunk_attention(q.to(DEV), torch.tensor(lens, device=DEV)).any()


def test_chunk_of_one_token_is_the_single_token_attention():
    st, o = _filled(4, 700, 128, "int8", seed=21)
    q = _rand((4 * 6, 1, 128), 9).view(4, 6, 128)
    for n, w, s in ((700, 0, 0), (333, 100, 5), (64, 0, 0)):
        one = st.attention(q.to(DEV), n, window=w, sinks=s).double()
        many = st.chunk_attention(q.to(DEV)[:, :, None], n, window=w, sinks=s)[:, :, 0].double()
        assert float((one - many).abs().max()) <= 1e-5 * float(one.abs().max())  # two float32 evaluations, each checked above


def test_chunk_query_layouts():
    """Token-major projections, padded heads, a shifted base, float64: the results of the plain layout, bit for bit."""
    st, _ = _filled(2, 200, 64, "e4m3", seed=5)
    q = _rand((2 * 4, 33, 64), 3, torch.bfloat16).view(2, 4, 33, 64).to(DEV)
    ref = st.chunk_attention(q, 150)
    token_major = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    padded = torch.zeros(2, 4, 33, 80, dtype=q.dtype, device=DEV)
    padded[..., 8:72] = q
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    strided = torch.zeros(2, 4, 33, 128, dtype=q.dtype, device=DEV)[..., ::2].copy_(q)
    for x in (token_major, padded[..., 8:72], odd, strided, q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(x, q) and torch.equal(st.chunk_attention(x, 150), ref)
    wide = st.chunk_attention(q.double(), 150)
    assert wide.dtype == torch.float32 and torch.equal(wide, st.chunk_attention(q.float(), 150))
    assert st.chunk_attention(q[:, :, :0], 150).shape == (2, 4, 0, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_chunk_what_a_query_does_not_see_does_not_count(dtype):
    """NaN codes, infinite and NaN scales in later tokens and between sinks and window leave a query as it is; the
    queries that see them are NaN."""
    G, T, n, D = 4, 100, 300, 128
    st, o = _filled(1, n, D, "e4m3", seed=31)
    q = _rand((G, T, D), 4, dtype).view(1, G, T, D).to(DEV)
    clean = {w: st.chunk_attention(q, n, window=w, sinks=3) for w in (0, 64)}
    at = 230  # place 230: queries from 30 on see it, with a window of 64 those from 30 to 93
    for what in ("v", "k"):
        bad, _ = _filled(1, n, D, "e4m3", seed=31)
        codes = (bad.v8 if what == "v" else bad.k8).view(torch.uint8)
        codes[0, at, 5] = 0x7F
        codes[0, at, 77] = 0xFF
        for w, last in ((0, T), (64, 94)):
            got = bad.chunk_attention(q, n, window=w, sinks=3)
            hit = torch.zeros(T, dtype=torch.bool, device=DEV)
            hit[at - (n - T):last] = True
            chans = torch.zeros(D, dtype=torch.bool, device=DEV)
            chans[[5, 77]] = True
            nan = (hit[:, None] & (chans if what == "v" else torch.ones_like(chans))).expand(1, G, T, D)
            assert torch.equal(got.isnan(), nan)
            assert torch.equal(got[~nan], clean[w][~nan])
    for value in (float("inf"), float("nan")):  # scales of the block from 256: queries from 56 on see it
        for s in ("k_scale", "v_scale"):
            bad, _ = _filled(1, n, D, "e4m3", seed=31)
            getattr(bad, s)[0, 4] = value
            got = bad.chunk_attention(q, n)
            assert torch.equal(got[:, :, :56], clean[0][:, :, :56])
            # an infinite score of either sign, or NaN; those of -inf alone leave the other tokens' attention
            dots = torch.matmul(q[0].double(), bad.k8[0, 256:].double().t().contiguous())
            seen = torch.arange(n - 256, device=DEV) <= torch.arange(T, device=DEV)[:, None] - 56
            finite = ((dots < 0) | ~seen).all(-1) if s == "k_scale" and value > 0 else ~seen.any(-1).expand(G, T)
            assert torch.equal(got[0].isfinite().all(-1), finite)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_chunk_blocks_of_any_scale(code):
    """Scales of K and V that differ by many powers of two, negative ones, zeros, weights far below the largest that carry the
    output because the large one's values are small."""
    G, T, n, D = 2, 40, 64 * 6, 128
    _, o = _filled(2, n, D, code, seed=41)
    o["vs"][0] *= np.float32(2.0) ** np.array([-90, 0, 30, -3, 0, 60], np.float32)
    o["vs"][1] *= np.float32(2.0) ** np.array([60, 0, -30, 3, 0, -60], np.float32)
    o["ks"][0, 1] *= -1
    o["vs"][1, 2] *= -1
    o["ks"][1, 3] = o["vs"][0, 1] = 0.0
    o["vs"][1, 4] = np.float32(1e-42)
    st = _from_numpy(o, code)
    for dtype in (torch.bfloat16, torch.float32):
        q = (_rand((2 * G, T, D), 8) * 4).to(dtype).view(2, G, T, D)
        _check_chunk(st.chunk_attention(q.to(DEV), n), q, o, code, [n, n], every=3)
    # one token takes nearly all of the weight and has no value
    st, o = _filled(1, n, D, code, seed=43)
    q = torch.zeros(1, 1, 3, D)
    q[..., 0] = 1.0
    o["k8"][0, :, 0] = 0
    o["k8"][0, 0, 0] = R.encode(np.array([100.0]), code)[0]
    o["ks"][0] = 1.0
    o["v8"][0, 0] = 0
    st = _from_numpy(o, code)
    for scale in (0.05, 0.15, 0.2):  # e^5, e^15, e^20 times the others' weight
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            _check_chunk(st.chunk_attention(q.to(dtype).to(DEV), n, scale=scale), q.to(dtype), o, code, [n], scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chunk_large_scores_and_queries_of_any_size(dtype):
    """Scores of +-2^10 to 2^40 (one token takes all), queries whose channels span the type, rows of zeros."""
    G, T, n, D = 2, 35, 200, 64
    st, o = _filled(1, n, D, "e4m3", seed=51)
    q = _rand((G, T, D), 2).view(1, G, T, D)
    for power in (10, 20, 40):
        big = (q * 2.0 ** power).to(dtype)
        got = st.chunk_attention(big.to(DEV), n).double().cpu().numpy()
        K, V = _values(o, "e4m3")
        z = np.einsum("gtd,nd->gtn", big[0].double().numpy(), K[0]) * D ** -0.5
        for g in range(G):
            for i in range(T):
                zz = np.sort(z[g, i, :n - T + i + 1])
                if zz[-1] - zz[-2] < 40 + 2.0 ** -20 * abs(zz[-1]):
                    continue  # the second largest counts too
                ref = V[0][int(z[g, i, :n - T + i + 1].argmax())]
                # the one weight as it is held, the value's product with it, the inverse of the sum and its product, the result
                assert np.allclose(got[0, g, i], ref, rtol=2.0 ** -BITS[dtype] + 4 * R.U + HALF[dtype], atol=1e-9)
    assert np.isfinite(got).all()
    tiny = q.clone()
    tiny[0, 0] *= 1e-30
    tiny[0, 0, :, 3] = 1.0
    tiny[0, 1] = 0.0
    tiny = tiny.to(dtype)
    _check_chunk(st.chunk_attention(tiny.to(DEV), n), tiny, o, "e4m3", [n], every=4)
    huge = (q.sign() * torch.finfo(dtype).max).to(dtype)
    assert st.chunk_attention(huge.to(DEV), n, scale=1e-38).isfinite().all()


# ----------------------------------------------------------------------------- windows with sinks, single tokens
@pytest.mark.parametrize("code, D, G", [("e4m3", 128, 4), ("int8", 64, 12), ("int8", 128, 9)])
@pytest.mark.parametrize("window, sinks, n", [(1, 1, 2), (64, 4, 333), (100, 64, 1000), (100, 65, 1000), (333, 300, 2000), (1500, 40, 2000),
                                              (64, 1999, 2000), (2000, 5, 2000), (128, 10 ** 12, 1999)])
def test_window_with_sinks(code, D, G, window, sinks, n):
    st, o = _filled(3, 2000, D, code, seed=61, garbage_behind=[n, n, n])
    K, V = _values(o, code)
    q = _rand((3, G, D), 5)
    sl = 2.0 ** -torch.arange(1.0, 3 * G + 1).view(3, G)
    lens = [n, n // 2, 1]
    for length, L in ((n, [n] * 3), (torch.tensor(lens, device=DEV), lens)):
        for cap, slopes in ((0.0, None), (20.0, sl)):
            got = st.attention(q.to(DEV), length, window=window, sinks=sinks, softcap=cap, slopes=None if slopes is None else slopes.to(DEV))
            for b in range(3):
                for g in range(G):
                    ref, tol = R.attention(q[b, g].double().numpy(), K[b], V[b], R.sees(L[b] - 1, L[b], window, sinks), L[b], D ** -0.5, cap,
                                           None if slopes is None else float(slopes[b, g]))
                    assert (np.abs(got[b, g].double().cpu().numpy() - ref) <= tol).all(), (b, g)


def test_window_with_sinks_in_splits():
    st, o = _filled(2, 30000, 128, "e4m3", seed=62)
    K, V = _values(o, "e4m3")
    q = _rand((2, 3, 128), 5)
    for n, window, sinks in ((30000, 9000, 8000), (25111, 20000, 70), (30000, 64, 29000)):
        for length in (n, torch.tensor([n, n - 64], device=DEV)):
            got = st.attention(q.to(DEV), length, window=window, sinks=sinks).double().cpu().numpy()
            for b in range(2):
                L = n if isinstance(length, int) else n - 64 * b
                for g in range(3):
                    ref, tol = R.attention(q[b, g].double().numpy(), K[b], V[b], R.sees(L - 1, L, window, sinks), L, 128 ** -0.5)
                    assert (np.abs(got[b, g] - ref) <= tol).all()


def test_sinks_leave_other_calls_as_they_are():
    """No sinks, or sinks that the window reaches: the bits of the call without the argument."""
    st, _ = _filled(2, 3000, 128, "e4m3", seed=63)
    q = _rand((2, 4, 128), 5).to(DEV)
    for n, window in ((3000, 0), (3000, 700), (100, 64), (3000, 3000)):
        ref = st.attention(q, n, window=window)
        assert torch.equal(ref, st.attention(q, n, window=window, sinks=0))
        if not window or window >= n:
            assert torch.equal(ref, st.attention(q, n, window=window, sinks=77))


def test_tokens_between_sinks_and_window_do_not_count():
    st, o = _filled(1, 1000, 128, "e4m3", seed=64)
    q = _rand((1, 4, 128), 5).to(DEV)
    ref = st.attention(q, 1000, window=100, sinks=10)
    for c in (st.k8, st.v8):
        c.view(torch.uint8)[0, 10:900] = 0x7F
    for s in (st.k_scale, st.v_scale):
        s[0, 1:14] = float("nan")  # blocks of tokens 64 .. 895
    assert torch.equal(ref, st.attention(q, 1000, window=100, sinks=10))
    many = st.chunk_attention(q[:, :, None], 1000, window=100, sinks=10)
    assert many.isfinite().all()


# ----------------------------------------------------------------------------- shared prefixes
def _check_shared(got, q, o, po, code, lens, plens, scale=None, softcap=0.0, slopes=None, rows=None):
    BH, G, D = q.shape
    H = po["k8"].shape[0]
    K, V = _values(o, code)
    PK, PV = _values(po, code)
    scale = D ** -0.5 if scale is None else scale
    got, qf = got.double().cpu().numpy(), q.double().cpu().numpy()
    for r in rows or range(BH):
        n, P = int(lens[r]), int(plens[r % H])
        # whole blocks, so that the bound's blocks are the stores'
        pad = -P % BLK
        k, v = (np.concatenate([p[r % H][:P], np.zeros((pad, D)), x[r][:n]]) for p, x in ((PK, K), (PV, V)))
        toks = np.concatenate([np.arange(P), P + pad + np.arange(n)])
        for g in range(G):
            s = None if slopes is None else float(slopes[r, g])
            bias = pad  # the padding is no distance: places are those of the joined row
            if s is not None and pad:
                k2, v2 = np.concatenate([PK[r % H][:P], K[r][:n]]), np.concatenate([PV[r % H][:P], V[r][:n]])
                ref, tol = R.many_attention(qf[r, g], k2, v2, np.arange(P + n), P + n, scale, softcap, s, 22, PARTS[q.dtype])
                tol = 2 * tol  # its blocks are shifted against the stores': one of them has parts of two
            else:
                ref, tol = R.many_attention(qf[r, g], k, v, toks, P + bias + n, scale, softcap, s, 22, PARTS[q.dtype])
            off = np.abs(got[r, g] - ref) - tol
            assert (off <= 0).all(), f"row {r} head {g}: {off.max():.3g} over {tol.max():.3g}"


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, H, G, P, n", [(1, 1, 1, 1, 1), (3, 2, 4, 200, 70), (9, 1, 5, 777, 130), (4, 3, 12, 64, 64)])
def test_shared(code, dtype, D, B, H, G, P, n):
    lens = [(n * (i % 4)) // 3 for i in range(B * H)]  # some rows without tokens of their own
    pst, po = _filled(H, P + 50, D, code, seed=71, garbage_behind=[P] * H)
    st, o = _filled(B * H, n, D, code, seed=72, garbage_behind=lens)
    q = _rand((B * H, G, D), 6, dtype)
    got = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, P)
    assert got.dtype == torch.float32
    _check_shared(got, q, o, po, code, lens, [P] * H)
    same = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, torch.tensor([P] * H, device=DEV))
    _check_shared(same, q, o, po, code, lens, [P] * H)


@pytest.mark.parametrize("softcap, slopes, scale", [(20.0, True, None), (0.0, True, 0.2), (3.0, False, -0.1)])
def test_shared_caps_and_slopes(softcap, slopes, scale):
    B, H, G, D = 5, 2, 3, 128
    lens, plens = [40, 0, 7, 64, 100, 3, 0, 0, 99, 1], [130, 64]
    pst, po = _filled(H, 192, D, "int8", seed=73)
    st, o = _filled(B * H, 100, D, "int8", seed=74)
    q = _rand((B * H, G, D), 6)
    sl = 2.0 ** -torch.arange(1.0, B * H * G + 1).fmod(9).view(B * H, G) if slopes else None
    got = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, torch.tensor(plens, device=DEV), scale=scale, softcap=softcap,
                              slopes=None if sl is None else sl.to(DEV))
    _check_shared(got, q, o, po, "int8", lens, plens, scale, softcap, sl)


@pytest.mark.parametrize("B, H, G, P, n, dtype", [(2, 1, 4, 30000, 3000, torch.float32), (33, 2, 4, 5000, 40, torch.bfloat16),
                                                  (70, 1, 1, 9999, 1200, torch.float16)])
def test_shared_in_splits(B, H, G, P, n, dtype):
    pst, po = _filled(H, P, 128, "e4m3", seed=75)
    st, o = _filled(B * H, n, 128, "e4m3", seed=76)
    q = _rand((B * H, G, 128), 6, dtype)
    rows = list(range(0, B * H, max(1, B * H // 5)))
    got = st.shared_attention(q.to(DEV), n, pst, P)
    _check_shared(got, q, o, po, "e4m3", [n] * B * H, [P] * H, rows=rows)
    lens = [n * i // (B * H) for i in range(B * H)]
    got = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, P)
    _check_shared(got, q, o, po, "e4m3", lens, [P] * H, rows=rows)


def test_shared_ends():
    """No prefix is the attention over the row's own tokens, no own tokens that over the prefix; nothing gives zeros."""
    st, _ = _filled(4, 300, 128, "e4m3", seed=77)
    pst, _ = _filled(2, 300, 128, "e4m3", seed=78)
    q = _rand((4, 4, 128), 6).to(DEV)
    close = lambda a, b: float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())  # noqa: E731
    assert close(st.shared_attention(q, 300, pst, 0), st.attention(q, 300))
    assert close(st.shared_attention(q, 0, pst, 222), torch.cat([pst.attention(q[2 * b:2 * b + 2], 222) for b in range(2)]))
    assert not st.shared_attention(q, 0, pst, 0).any()
    zero = torch.zeros(4, dtype=torch.int32, device=DEV)
    assert not st.shared_attention(q, zero, pst, zero[:2]).any()


# ----------------------------------------------------------------------------- tiles of eight waves, shares
@pytest.mark.parametrize("code, dtype, D", [("e4m3", torch.bfloat16, 128), ("int8", torch.float16, 64), ("e4m3", torch.float16, 64),
                                            ("int8", torch.bfloat16, 128), ("e4m3", torch.float32, 128)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (900, 70), (1000, 0)])
def test_chunk_of_many_queries(code, dtype, D, window, sinks):
    """2400 queries of a row, the last tile not full, rows of one length and of many: tiles of eight waves for 16-bit queries, of
    four for float32 ones and with a cap."""
    BH, G, T, n = 6, 8, 300, 1700
    lens = [1700, 1333, 290, 0, 301, 64]
    st, o = _filled(BH, n, D, code, seed=15, garbage_behind=lens)
    q = _rand((BH * G, T, D), 16, dtype).view(BH, G, T, D)
    ragged = torch.tensor(lens, device=DEV)
    _check_chunk(st.chunk_attention(q.to(DEV), ragged, window=window, sinks=sinks), q, o, code, lens, window, sinks, every=59)
    _check_chunk(st.chunk_attention(q.to(DEV), ragged, window=window, sinks=sinks, softcap=20.0), q, o, code, lens, window, sinks,
                 softcap=20.0, every=83)
    st, o = _filled(BH, n, D, code, seed=17)
    _check_chunk(st.chunk_attention(q.to(DEV), n, window=window, sinks=sinks), q, o, code, [n] * BH, window, sinks, every=71)


@pytest.mark.parametrize("B, H, G, P, n, dtype", [(520, 2, 4, 3800, 20, torch.bfloat16), (65, 4, 4, 16300, 3, torch.float16),
                                                  (300, 1, 7, 9000, 10, torch.bfloat16)])
def test_shared_by_many(B, H, G, P, n, dtype):
    pst, po = _filled(H, P, 64, "int8", seed=91)
    st, o = _filled(B * H, n, 64, "int8", seed=92)
    q = _rand((B * H, G, 64), 6, dtype)
    rows = list(range(0, B * H, B * H // 9)) + [B * H - 1]
    lens = [n * (i % 3) // 2 for i in range(B * H)]
    for length, prefix_length in ((torch.tensor(lens, device=DEV), P), (torch.tensor(lens, device=DEV), torch.tensor([P] * H, device=DEV))):
        got = st.shared_attention(q.to(DEV), length, pst, prefix_length)
        _check_shared(got, q, o, po, "int8", lens, [P] * H, rows=rows)
    sl = torch.full((B * H, G), 2.0 ** -7)
    got = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, P, softcap=10.0, slopes=sl.to(DEV))
    _check_shared(got, q, o, po, "int8", lens, [P] * H, softcap=10.0, slopes=sl, rows=rows)


@pytest.mark.parametrize("BH, G, T, n, at", [(1, 2, 3, 30011, 29000), (1, 2, 3, 30011, 7), (6, 8, 300, 1700, 1500), (2, 4, 20, 9000, 8999)])
def test_a_nan_in_one_of_many_shares(BH, G, T, n, at):
    """A NaN code of V, or a scale of V that is infinite, makes the channels NaN of the queries that see it, and no others."""
    q = _rand((BH * G, T, 128), 4, torch.bfloat16).view(BH, G, T, 128).to(DEV)
    st, _ = _filled(BH, n, 128, "e4m3", seed=33)
    clean = st.chunk_attention(q, n)
    sees = torch.arange(n - T, n, device=DEV) >= at
    st.v8.view(torch.uint8)[-1, at, 41] = 0xFF
    got = st.chunk_attention(q, n)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[-1, :, sees, 41] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])
    st.v_scale[-1, at // BLK] = float("inf")
    got = st.chunk_attention(q, n)
    nan[-1, :, torch.arange(n - T, n, device=DEV) >= at // BLK * BLK] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("code, D", [("e4m3", 128), ("int8", 64), ("int8", 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_caps_that_bind(code, D, dtype):
    """Scores of many times the cap and near it, in tiles of one wave and of four, few and many of a block."""
    n = 333
    st, o = _filled(2, n, D, code, seed=95)
    for G, T in ((2, 5), (3, 50)):
        q = _rand((2 * G, T, D), 7, dtype).view(2, G, T, D)
        q[:, :, ::3] *= 2.0 ** -6
        for scale, cap in ((2.0, 5.0), (0.5, 3.0), (-1.0, 12.0)):
            got = st.chunk_attention(q.to(DEV), n, scale=scale, softcap=cap)
            _check_chunk(got, q, o, code, [n, n], scale=scale, softcap=cap, every=7)


@pytest.mark.parametrize("code, D", [("e4m3", 128), ("int8", 64)])
@pytest.mark.parametrize("power", [-17, -20, -28, -40])
def test_small_channels_of_float32_queries(code, D, power):
    """Channels of 2^-17 to 2^-40 of the query's largest, which meets K's zeros, decide the scores: with two f16 parts alone those
    would be off by 2^-8 of themselves and more."""
    n = 200
    _, o = _filled(2, n, D, code, seed=97)
    o["k8"][:, :, 3] = 0
    o["ks"] *= np.float32(2.0 ** -power)
    st = _from_numpy(o, code)
    for G, T in ((2, 5), (2, 40), (3, 70)):
        q = _rand((2 * G, T, D), 8).view(2, G, T, D) * 2.0 ** power
        q[..., 3] = 1.0
        q[:, :, 2::3, 3] = 0.0  # some queries without the large channel
        _check_chunk(st.chunk_attention(q.to(DEV), n), q, o, code, [n, n], every=6)


@pytest.mark.parametrize("seed", range(10))
def test_chunks_are_single_tokens_at_many_shapes(seed):
    """Rows from 1 to 600, 1 to 33 heads, chunks from one token on, windows, sinks, caps, biases, lengths of each row or of all: a
    chunk's tokens against the single-token attention, another kernel.  Both are within the oracle's bound; here with A the largest
    |q| |K| scale of any token, and |V| <= its largest for the weighted mean of it: (4 D + 64) 2 U A for the two chains of D products
    (of three parts in float32) and what follows, the joins, the weights' bits and their ends, half a step of the output."""
    rng = np.random.default_rng(1000 + seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pick = lambda *x: x[rng.integers(len(x))]  # noqa: E731
    for _ in range(12):
        D, code, dtype = pick(64, 128), pick("e4m3", "int8"), pick(torch.bfloat16, torch.float16, torch.float32)
        BH, G, T = pick(1, 2, 3, 5, 17, 70, 260, 600), pick(1, 2, 3, 4, 7, 8, 12, 33), pick(1, 2, 4, 5, 8, 9, 31, 33, 64, 100, 257, 700)
        T = max(1, min(T, 40000 // (BH * G)))
        n = max(1, min(int(2 ** rng.uniform(0, 14)), 1000000 // BH))
        cap = n + int(rng.integers(130))
        window = pick(0, 0, 1, 63, 64, 65, 500)
        kw = dict(window=window, sinks=pick(0, 1, 64, 100) if window else 0, softcap=pick(None, None, 30.0, 4.0))
        slopes = torch.exp2(-8 * torch.rand(BH, G, device=DEV, generator=gen)) if rng.random() < 0.3 else None
        case = (D, code, str(dtype), BH, G, T, n, cap, kw, slopes is not None)
        st = RowStore8.empty(BH, cap, CODES[code], D, DEV)
        K, V = torch.randn(2, BH, cap, D, device=DEV, generator=gen)
        st.write(K, V)
        lens = torch.full((BH,), n, dtype=torch.int32, device=DEV)
        length = n
        if rng.random() < 0.5:
            length = lens = torch.from_numpy(rng.integers(0, n + 1, BH).astype(np.int32)).to(DEV)
        q = torch.randn(BH, G, T, D, device=DEV, generator=gen).to(dtype)
        got = st.chunk_attention(q, length, slopes=slopes, **kw).double()
        K, V = st.read(0, cap, torch.float32)
        big = float(V.abs().max())
        A = float(torch.bmm(q.float().abs().view(BH, G * T, D), K.abs().transpose(1, 2).contiguous()).max()) * D ** -0.5
        rel = 2 * (4 * D + 64) * R.U * A + 2 * (n / 8 + 64) * R.U + 2 * 2.0 ** -BITS[dtype] + 2.0 ** -20 + n * 2.0 ** -33
        for i in {0, T // 2, T - 1}:
            seen = lens - (T - 1 - i)
            one = st.attention(q[:, :, i].contiguous(), seen.clamp(min=0), slopes=slopes, **kw).double()
            one[seen <= 0] = 0
            off = (got[:, :, i] - one).abs() - rel * big - one.abs().clamp(min=2.0 ** -14) * HALF[dtype]
            assert float(off.max()) <= 0, (case, i)


def test_calls_with_and_without_a_cap_in_turn():
    """The same shapes with and without a cap take other tiles, and workspaces of one size."""
    st, _ = _filled(6, 1700, 128, "e4m3", seed=96)
    q = _rand((48, 300, 128), 6, torch.bfloat16).view(6, 8, 300, 128).to(DEV)
    lens = torch.tensor([1700, 1300, 900, 500, 310, 300], dtype=torch.int32, device=DEV)
    far = 1e29  # a cap that no score feels
    plain, capped = st.chunk_attention(q, lens), st.chunk_attention(q, lens, softcap=far)
    assert torch.equal(plain, capped)
    zeros = torch.zeros(8, device=DEV)
    biased = st.chunk_attention(q, lens, slopes=zeros)
    # both are off by half a step of bf16 at most, from values that are off by less
    assert float((biased.float() - plain.float()).abs().max()) <= 2 ** -7 * float(plain.float().abs().max())
    for _ in range(2):
        assert torch.equal(st.chunk_attention(q, lens), plain) and torch.equal(st.chunk_attention(q, lens, slopes=zeros), biased)


# ----------------------------------------------------------------------------- calls
def test_calls_repeat_bit_for_bit_on_any_stream():
    st, _ = _filled(4, 5000, 128, "e4m3", seed=81)
    pst, _ = _filled(2, 5000, 128, "e4m3", seed=82)
    q4 = _rand((8, 8, 128), 6, torch.bfloat16).view(4, 2, 8, 128).to(DEV)
    q3 = q4[:, :, 0].contiguous()
    calls = [lambda: st.chunk_attention(q4, 5000), lambda: st.shared_attention(q3, 3000, pst, 5000),
             lambda: st.attention(q3, 5000, window=900, sinks=70)]
    torch.cuda.synchronize()
    for f in calls:
        ref = f()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = f()
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(ref, other) and torch.equal(ref, f())


def test_captured_calls_follow_their_lengths():
    """Graphs of each call, replayed in turn with lengths that change between replays, equal the eager calls."""
    st, _ = _filled(4, 5000, 128, "e4m3", seed=83)
    pst, _ = _filled(2, 3000, 128, "e4m3", seed=84)
    q4 = _rand((8, 8, 128), 6, torch.bfloat16).view(4, 2, 8, 128).to(DEV)
    q3 = q4[:, :, 0].contiguous()
    lens = torch.full((4,), 5000, dtype=torch.int32, device=DEV)
    plens = torch.full((2,), 3000, dtype=torch.int32, device=DEV)
    calls = [lambda: st.chunk_attention(q4, lens), lambda: st.shared_attention(q3, lens, pst, plens),
             lambda: st.attention(q3, lens, window=900, sinks=70), lambda: st.chunk_attention(q4, lens, window=333, sinks=4)]
    for f in calls:
        f()
    torch.cuda.synchronize()
    graphs = []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    for L, P in (([5000, 1, 64, 0], [3000, 100]), ([7, 4999, 2500, 5000], [0, 1]), ([5000] * 4, [3000] * 2)):
        lens.copy_(torch.tensor(L))
        plens.copy_(torch.tensor(P))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (g, out), f in zip(graphs, calls):
            assert torch.equal(out, f())


def test_offsets_past_32_bits():
    """Rows of 2^24 + 100 tokens: codes of the second one begin past 2^31 bytes, its last tokens past 2^32."""
    cap, D = (1 << 24) + 100, 128
    st = RowStore8.empty(2, cap, torch.int8, D, DEV)
    K, V = _rand((2, 300, D), 1, torch.bfloat16), _rand((2, 300, D), 2, torch.bfloat16)
    st.write(K.to(DEV), V.to(DEV), cap - 300)
    o = {"k8": np.zeros((2, 384, D), np.uint8), "v8": np.zeros((2, 384, D), np.uint8)}
    o["ks"], o["vs"] = np.zeros((2, 2, 6), np.float32)
    lead = (cap - 300) % BLK
    R.write(o, _f32(K), _f32(V), lead, "int8")
    n, window = lead + 300, 200
    q = _rand((2 * 2, 20, D), 3, torch.bfloat16).view(2, 2, 20, D)
    got = st.chunk_attention(q.to(DEV), cap, window=window)
    _check_chunk(got, q, o, "int8", [n, n], window, every=3)
    one = st.attention(q[:, :, -1].contiguous().to(DEV), cap, window=window, sinks=0)
    assert float((one - got[:, :, -1].float()).abs().max()) <= 2.0 ** -7 * float(one.abs().max())


def test_refusals():
    st, _ = _filled(4, 100, 128, "e4m3")
    other, _ = _filled(3, 100, 128, "e4m3")
    ints, _ = _filled(2, 100, 128, "int8")
    short, _ = _filled(2, 100, 64, "e4m3")
    pst, _ = _filled(2, 100, 128, "e4m3")
    q = torch.zeros(4, 2, 8, 128, dtype=torch.bfloat16, device=DEV)
    q3 = q[:, :, 0].contiguous()
    for bad in (q[:3], q[..., :64], q3, q[:, :0], q.cpu()):
        with pytest.raises(ValueError):
            st.chunk_attention(bad, 100)
    for kw in (dict(length=101), dict(length=-1), dict(length=100, window=-1), dict(length=100, sinks=-1), dict(length=100, softcap=-1.0),
               dict(length=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(length=torch.zeros(4, device=DEV)), dict(length=1 << 63)):
        with pytest.raises(ValueError):
            st.chunk_attention(q, **kw)
    with pytest.raises(ValueError):
        st.attention(q3, 100, window=10, sinks=-1)
    for prefix in (other, ints, short, None, q3):
        with pytest.raises(ValueError):
            st.shared_attention(q3, 100, prefix, 100)
    for kw in (dict(length=101, prefix_length=5), dict(length=5, prefix_length=101), dict(length=5, prefix_length=-1),
               dict(length=5, prefix_length=torch.zeros(4, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            st.shared_attention(q3, prefix=pst, **kw)


# ----------------------------------------------------------------------------- what only some of a wave's queries see
# one wave's tiles, four waves' and eight waves' (BH, G, T, n): a block's edge lies inside a wave of each
FORMS = [(2, 4, 8, 197), (1, 2, 3, 30018), (1, 4, 100, 310), (8, 8, 300, 1241)]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("BH, G, T, n", FORMS)
def test_a_scale_of_k_that_is_not_finite_reaches_only_queries_that_see_it(BH, G, T, n, dtype, value):
    D = 128
    q = _rand((BH * G, T, D), 4, dtype).view(BH, G, T, D).to(DEV)
    st, o = _filled(BH, n, D, "e4m3", seed=34)
    edge = (n - T // 2) // BLK * BLK  # queries before this place do not see the block that it begins
    assert n - T < edge < n - 1
    clean = st.k_scale[:, edge // BLK].clone()
    st.k_scale[:, edge // BLK] = value
    before = edge - (n - T)
    got = st.chunk_attention(q, n)
    if value != value:
        assert got[:, :, before:].isnan().all()
    _check_chunk(got[:, :, :before], q[:, :, :before], o, "e4m3", [edge] * BH, every=max(1, before // 4))
    _check_chunk(got[:, :, before - 1:before], q[:, :, before - 1:before], o, "e4m3", [edge] * BH)
    # queries whose window has passed the block before that place
    st.k_scale[:, edge // BLK] = clean
    st.k_scale[:, edge // BLK - 1] = value
    behind = n - T // 2
    window, first, last = behind - edge + 1, max(edge - BLK - (n - T), 0), behind - (n - T)
    got = st.chunk_attention(q, n, window=window, sinks=3)
    if value != value:
        assert got[:, :, first:last].isnan().all()
    _check_chunk(got[:, :, :first], q[:, :, :first], o, "e4m3", [n - T + first] * BH, window, 3, every=max(1, first // 4))
    _check_chunk(got[:, :, last:], q[:, :, last:], o, "e4m3", [n] * BH, window, 3, every=max(1, (T - last) // 4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("BH, G, T", [(1, 1, 1), (2, 4, 8), (1, 4, 40), (8, 8, 300)])
def test_a_block_of_nan_values_makes_nan(BH, G, T, dtype):
    """V that is NaN throughout a block, or NaN among zeros, has the smallest scale there is: NaN all the same for the queries that
    see it, wherever the block lies, as for single tokens."""
    D, n = 128, 990 + T
    q = _rand((BH * G, T, D), 4, dtype).view(BH, G, T, D).to(DEV)
    K, V = _rand((BH, n, D), 1), _rand((BH, n, D), 2)
    for zeros in (False, True):
        for block in (0, 5, 14):
            bad = V.clone()
            bad[-1, block * BLK:(block + 1) * BLK] = 0.0 if zeros else float("nan")
            bad[-1, block * BLK + 7, 33] = float("nan")
            st = RowStore8.empty(BH, n, torch.float8_e4m3fn, D, DEV)
            st.write(K.to(DEV), bad.to(DEV))
            nan = torch.zeros(BH, G, T, D, dtype=torch.bool)
            nan[-1, :, :, slice(33, 34) if zeros else slice(None)] = True
            assert torch.equal(st.chunk_attention(q, n).isnan().cpu(), nan)
            last = q[:, :, -1].contiguous()
            assert torch.equal(st.attention(last, n).isnan().cpu(), nan[:, :, -1])
            own = RowStore8.empty(BH * T, 1, torch.float8_e4m3fn, D, DEV)
            got = own.shared_attention(q.permute(2, 0, 1, 3).reshape(BH * T, G, D), 0, st, n)
            assert torch.equal(got.isnan().cpu().view(T, BH, G, D), nan.permute(2, 0, 1, 3))


# ----------------------------------------------------------------------------- scores far from zero
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("BH, G, T", [(1, 2, 5), (2, 4, 40), (8, 8, 300)])
@pytest.mark.parametrize("power", [7, 10, 14, 17, 20, 24, 26, 30])
def test_equal_scores_weigh_the_same_in_blocks_of_other_scales(dtype, BH, G, T, power):
    """Tokens of one score, 2^power, in blocks whose scales of V differ, above all others': the mean of their values.

    Their weights are one number, each held with an error e of 2^-bits at most (half a step of what it is held in) and divided by a sum
    of those: 2 e of the mean |v|.  A factor of V that goes into the exponent of an 11-bit weight adds half a step of that exponent,
    below 512: ln 2 2^-16, and steps of log2 and exp2 and of the products: together below 2^-15, for 22 bits 2^-21.  (At 2^7 the
    others' weights are below e^-128 of it, which is nothing.)"""
    D, n = 128, 64 * 18 + T
    rng = np.random.default_rng(power)
    o = {"k8": np.zeros((BH, n, D), np.uint8), "v8": rng.integers(1, 0x78, (BH, n, D), dtype=np.uint8)}
    o["ks"] = np.full((BH, -(-n // BLK)), 2.0 ** (power - 10), np.float32)
    o["vs"] = np.exp2(rng.uniform(-4, 4, o["ks"].shape)).astype(np.float32)
    top = [np.sort(rng.choice(64 * 18, 7, replace=False)) for _ in range(BH)]
    for b in range(BH):
        o["k8"][b, top[b], 0] = R.encode(np.array([64.0]), "e4m3")[0]
    st = _from_numpy(o, "e4m3")
    q = torch.zeros(BH, G, T, D, dtype=dtype)
    q[..., 0] = 16.0
    V = _values(o, "e4m3")[1]

    def check(got, bits, half):
        for b in range(BH):
            v = V[b, top[b]]
            tol = 2 * (2.0 ** -bits + (2.0 ** -15 if bits == 11 else 2.0 ** -21)) * np.abs(v).mean(0)
            off = np.abs(got[b].double().cpu().numpy() - v.mean(0)) - tol - half * (np.abs(v.mean(0)) + tol)
            assert (off <= 0).all(), f"row {b}: {off.max():.3g} over {tol.max():.3g}"

    check(st.chunk_attention(q.to(DEV), n, scale=1.0), BITS[dtype], HALF[dtype])
    own, _ = _filled(BH * T, 5, D, "e4m3")  # its scores are far smaller
    own.k_scale.mul_(2.0 ** -20)
    got = own.shared_attention(q.permute(2, 0, 1, 3).reshape(BH * T, G, D).to(DEV), 5, st, n, scale=1.0)
    check(got.view(T, BH, G, D).permute(1, 2, 0, 3), 22, 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("BH, G, T", [(1, 2, 5), (1, 4, 40), (8, 8, 300)])
def test_shares_of_scores_on_both_sides_of_a_power_of_two(dtype, BH, G, T):
    """Scores of 2^26 - 8 in most blocks and of 2^26 + 16 in one (in units of log 2, as float32 has them): steps of 4 and of 8, where the
    waves' and shares' maxima are apart by what is no multiple of the steps.  What the lower ones weigh together, 2^-24 each, is seen
    in a channel of their own."""
    D, n = 128, 64 * 20 + T
    L = np.float32(1.44269504088896340736)
    s = 4 * np.arange((1 << 26) // 6, (1 << 26) // 5, dtype=np.int64)
    r = s.astype(np.float32) * L
    low, high = (int(s[np.flatnonzero(r == np.float32(2.0 ** 26 + x))[0]]) for x in (-8, 16))
    o = {"k8": np.zeros((BH, n, D), np.uint8), "v8": np.zeros((BH, n, D), np.uint8)}
    o["ks"] = np.full((BH, -(-n // BLK)), 2.0 ** 10, np.float32)
    o["vs"] = np.ones_like(o["ks"])
    one = R.encode(np.array([1.0]), "e4m3")[0]
    bits = lambda x: np.array([one if x >> j & 1 else 0 for j in range(2, 26)], np.uint8)  # noqa: E731
    o["k8"][:, :, :24] = bits(low)
    o["v8"][:, :, 3] = one
    at = 64 * 7 + 9
    o["k8"][:, at, :24] = bits(high)
    o["v8"][:, at] = 0
    o["v8"][:, at, 5] = one
    st = _from_numpy(o, "e4m3")
    q = torch.zeros(BH, G, T, D)
    q[..., :24] = torch.exp2(torch.arange(2.0, 26.0) - 10)
    q = q.to(dtype)
    got = st.chunk_attention(q.to(DEV), n, scale=1.0).double().cpu()
    low_ones = (n - T + torch.arange(T, dtype=torch.float64)) * 2.0 ** -24  # of the tokens up to the query's all but one
    # the weights are powers of two; sums of n of them round 2^-24 each at most, the result half a step of its type
    for ref, channel in ((low_ones / (1 + low_ones), 3), (1 / (1 + low_ones), 5)):
        off = (got[..., channel] - ref).abs()
        assert (off <= ref * (n * R.U) + torch.maximum(ref * HALF[dtype], torch.tensor(FLOOR[dtype], dtype=torch.float64))).all()


def test_a_prefix_without_rows_is_refused():
    st, _ = _filled(4, 100, 128, "e4m3")
    none = RowStore8.empty(0, 100, torch.float8_e4m3fn, 128, DEV)
    with pytest.raises(ValueError):
        st.shared_attention(torch.zeros(4, 2, 128, device=DEV), 100, none, 100)


def test_scales_that_are_not_finite_are_refused():
    st, _ = _filled(4, 100, 128, "e4m3")
    pst, _ = _filled(2, 100, 128, "e4m3")
    q = torch.zeros(4, 2, 8, 128, dtype=torch.bfloat16, device=DEV)
    for scale in (float("nan"), float("inf"), -float("inf"), 3e38, 1e39):
        with pytest.raises(ValueError):
            st.chunk_attention(q, 100, scale=scale)
        with pytest.raises(ValueError):
            st.shared_attention(q[:, :, 0].contiguous(), 100, pst, 100, scale=scale)


def test_biased_rows_behind_whole_blocks_of_a_prefix():
    """With a bias and prefixes that end with a block, the joined row has the stores' blocks, so that the bound is the oracle's own."""
    B, H, G, D = 5, 2, 3, 128
    lens, plens = [40, 0, 7, 64, 100, 3, 0, 0, 99, 1], [128, 64]
    for code in ("int8", "e4m3"):
        pst, po = _filled(H, 192, D, code, seed=173)
        st, o = _filled(B * H, 100, D, code, seed=174)
        sl = 2.0 ** -torch.arange(1.0, B * H * G + 1).fmod(9).view(B * H, G)
        for dtype in (torch.bfloat16, torch.float32):
            q = _rand((B * H, G, D), 6, dtype)
            for softcap, scale in ((20.0, None), (0.0, 0.2)):
                got = st.shared_attention(q.to(DEV), torch.tensor(lens, device=DEV), pst, torch.tensor(plens, device=DEV), scale=scale,
                                          softcap=softcap, slopes=sl.to(DEV))
                _check_shared(got, q, o, po, code, lens, plens, scale, softcap, sl)


def test_capped_plain_and_biased_calls_in_turn():
    """The same shapes with a cap, without one and with a bias take kernels and tiles of their own: each call repeats its own bits with
    the others in between, and a cap that no score feels changes a result by roundings alone."""
    st, o = _filled(6, 1700, 128, "e4m3", seed=96)
    q = _rand((48, 300, 128), 6, torch.bfloat16).view(6, 8, 300, 128)
    lens = [1700, 1300, 900, 500, 310, 300]
    on, length = q.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    zeros = torch.zeros(8, device=DEV)
    calls = [dict(), dict(softcap=1e4), dict(slopes=zeros), dict(softcap=5.0), dict(softcap=1e4, slopes=zeros)]
    first = [st.chunk_attention(on, length, **kw) for kw in calls]
    assert not torch.equal(first[0], first[3])
    for kw, ref in zip(calls, first):
        _check_chunk(ref, q, o, "e4m3", lens, softcap=kw.get("softcap", 0.0), slopes=torch.zeros(6, 8) if "slopes" in kw else None, every=97)
    for _ in range(3):
        for kw, ref in zip(calls, first):
            assert torch.equal(st.chunk_attention(on, length, **kw), ref)
