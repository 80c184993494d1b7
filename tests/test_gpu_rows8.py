"""The 8-bit K/V row store on the GPU against its oracle: codes, scales and values bit
for bit; attention within the oracle's bound of a float32 evaluation."""
import numpy as np
import pytest
import torch

from fathom_amd import bitplane as bp
from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BLK = 64


def _rand(shape, seed, dtype=torch.float32, spread=1.0):
    """Normal rows with lognormal channel scales."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, shape[2], generator=g))
    return x.to(dtype)


def _f32(x):
    return x.float().numpy()


def _garbage(BH, cap, D, code, seed=99):
    """A store of arbitrary bytes (e4m3 NaN among them) and scales of every kind, and its numpy copy."""
    rng = np.random.default_rng(seed)
    o = {"k8": rng.integers(0, 256, (BH, cap, D), dtype=np.uint8), "v8": rng.integers(0, 256, (BH, cap, D), dtype=np.uint8)}
    nblk = -(-cap // BLK)
    for s in ("ks", "vs"):
        o[s] = np.where(rng.random((BH, nblk)) < 0.5, np.float32(np.nan), rng.random((BH, nblk), dtype=np.float32) * 3)
        o[s] = o[s].astype(np.float32)
    return _from_numpy(o, code), o


def _from_numpy(o, code):
    k8, v8 = (torch.from_numpy(o[n].copy()).to(DEV).view(CODES[code]) for n in ("k8", "v8"))
    return RowStore8(k8, v8, torch.from_numpy(o["ks"].copy()).to(DEV), torch.from_numpy(o["vs"].copy()).to(DEV))


def _empty(BH, cap, D, code):
    o = {"k8": np.zeros((BH, cap, D), np.uint8), "v8": np.zeros((BH, cap, D), np.uint8),
         "ks": np.zeros((BH, -(-cap // BLK)), np.float32), "vs": np.zeros((BH, -(-cap // BLK)), np.float32)}
    return RowStore8.empty(BH, cap, CODES[code], D, DEV), o


def _same(st, o, code, nan_payload=False):
    for t, n in ((st.k8, "k8"), (st.v8, "v8")):
        got, ref = t.view(torch.uint8).cpu().numpy(), o[n]
        if code == "e4m3" and not nan_payload:  # NaN of either sign
            got, ref = np.where(got & 0x7F == 0x7F, 0x7F, got), np.where(ref & 0x7F == 0x7F, 0x7F, ref)
        bad = got != ref
        assert not bad.any(), f"{n}: {int(bad.sum())} codes differ, first at {np.argwhere(bad)[0]}"
    for t, n in ((st.k_scale, "ks"), (st.v_scale, "vs")):
        assert np.array_equal(t.cpu().numpy().view(np.uint32), o[n].view(np.uint32)), n


# ----------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T, pos, cap", [(1, 0, 1), (1, 63, 100), (1, 64, 100), (2, 63, 333), (64, 0, 64), (63, 1, 64),
                                         (200, 37, 333), (333, 0, 333), (129, 204, 333)])
def test_write_bit_exact(code, dtype, D, T, pos, cap):
    st, o = _garbage(3, cap, D, code)
    o["ks"][0], o["vs"][1] = 1e-4, 2e-3  # small scales that have to grow; the others hold NaN or any size
    st = _from_numpy(o, code)
    K, V = _rand((3, T, D), 1, dtype), _rand((3, T, D), 2, dtype, 2.0)
    st.write(K.to(DEV), V.to(DEV), pos)
    R.write(o, _f32(K), _f32(V), pos, code)
    _same(st, o, code)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_write_edge_values(code, dtype):
    D, T = 128, 5 * 64
    big = torch.finfo(dtype).max
    K = _rand((2, T, D), 3).clamp(-100, 100)
    K[0, :64] = 0.0
    K[0, 64:128, :5] = torch.tensor([float("inf"), -float("inf"), float("nan"), big, -big])
    K[0, 128:192] = float("nan")
    K[0, 192:256] = float("inf")
    K[0, 256:] *= torch.finfo(dtype).tiny
    K[1, :64] = -0.0
    K[1, 64:128] = torch.arange(64 * 128).view(64, 128) % 255 - 127.0      # every int8 code, scale 1
    K[1, 128:192] = (torch.arange(64 * 128).view(64, 128) % 509 - 254) / 2  # ties
    K[1, 192:256] = torch.from_numpy(R.E4M3[:127]).float().repeat(65)[:64 * 128].view(64, 128)
    K = K.to(dtype)
    V = K.flip(1)
    st, o = _empty(2, T, D, code)
    st.write(K.to(DEV), V.to(DEV))
    R.write(o, _f32(K), _f32(V), 0, code)
    _same(st, o, code)
    got = st.read(0, T, torch.float32)[0].cpu().numpy()
    ref = R.values(o["k8"], o["ks"], code)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, ref.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
def test_growth_token_by_token(code, D):
    """Blocks that grow token by token, each larger than the last, equal the oracle after every write, and the roundings
    that add up stay within one last step (int8) or half a step of the format (e4m3, normal codes)."""
    n = 130
    x = _rand((2, n, D), 4, spread=0.3) * torch.exp(torch.linspace(0, 5, n))[None, :, None]
    st, o = _empty(2, 200, D, code)
    for t in range(n):
        xt = x[:, t:t + 1]
        st.write(xt.to(DEV), -xt.to(DEV), t)
        R.write(o, _f32(xt), _f32(-xt), t, code)
        if t % 16 == 15 or t == n - 1:
            _same(st, o, code)
    v = R.values(o["k8"], o["ks"], code)[:, :n]
    s = np.repeat(o["ks"], BLK, 1)[:, :n, None].astype(np.float64)
    err = np.abs(v - x.double().numpy())
    if code == "int8":
        assert (err <= s * (1 + 1e-5)).all()
    else:
        # half a step: 2^-4 of the value or, where a code is subnormal, each of the roundings half of 2^-9 of a scale that doubles
        assert (err <= np.maximum(np.abs(x.double().numpy()) * 2.0 ** -4, s * 2.0 ** -9) * (1 + 1e-5)).all()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_write_ragged_places(code):
    """Rows at places of their own; rows whose tokens do not all fit stay as they are."""
    BH, cap, T, D = 7, 500, 90, 128
    st, o = _garbage(BH, cap, D, code)
    pos = np.array([0, 409, 410, 411, -1, 64, 2 ** 31 - 1])
    K, V = _rand((BH, T, D), 5, torch.bfloat16), _rand((BH, T, D), 6, torch.bfloat16)
    for p in (torch.from_numpy(pos).to(DEV), torch.from_numpy(pos.astype(np.int32)).to(DEV)):
        st.write(K.to(DEV), V.to(DEV), p)
        R.write(o, _f32(K), _f32(V), pos, code)
        _same(st, o, code)
    st.write(K.to(DEV), V.to(DEV), torch.tensor([2 ** 32 + 5] * BH, device=DEV))  # beyond int32: fits nowhere
    _same(st, o, code)


def test_write_strided_views():
    """[B, T, H, D] projections, slices of a wider tensor, and rows at odd addresses."""
    B, H, T, D = 2, 3, 70, 64
    qkv = _rand((B * T, 1, H * 3 * D + 24), 7, torch.float16).view(B, T, -1).to(DEV)
    K = qkv[..., H * D:2 * H * D].unflatten(2, (H, D)).transpose(1, 2)  # [B, H, T, D]
    V = qkv[..., 2 * H * D + 1:3 * H * D + 1].unflatten(2, (H, D)).transpose(1, 2)  # at an odd element
    for b in range(B):
        st, o = _empty(H, 100, D, "int8")
        st.write(K[b], V[b], 11)
        R.write(o, _f32(K[b].cpu()), _f32(V[b].cpu()), 11, "int8")
        _same(st, o, "int8")
    st, o = _empty(H, 100, D, "int8")
    every = K[0].transpose(1, 2).contiguous().transpose(1, 2)  # rows not dense
    st.write(every, K[0][:1].expand(H, T, D), 0)
    R.write(o, _f32(K[0].cpu()), _f32(K[0][:1].expand(H, T, D).cpu()), 0, "int8")
    _same(st, o, "int8")
    one = qkv.view(-1)[4:4 + 203 * 3].view(1, 3, 203)  # a single row and token, with strides that are no multiple of 16 bytes
    st1, o1 = _empty(1, 100, D, "int8")
    for x in (one[:, 1:2, 4:68], one[:, :1, 20:84], one[:, ::2, 4:68]):
        st1.write(x, x, 9)
        R.write(o1, _f32(x.cpu()), _f32(x.cpu()), 9, "int8")
        _same(st1, o1, "int8")
    st.write(K[0].double(), V[0].double(), 0)  # other types go through float32
    R.write(o, _f32(K[0].cpu()), _f32(V[0].cpu()), 0, "int8")
    _same(st, o, "int8")


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_read(code, D, dtype):
    BH, cap = 3, 333
    st, o = _empty(BH, cap, D, code)
    K, V = _rand((BH, cap, D), 8), _rand((BH, cap, D), 9)
    st.write(K.to(DEV), V.to(DEV))
    R.write(o, _f32(K), _f32(V), 0, code)
    ref = {n: torch.from_numpy((R.decode(o[c], code).astype(np.float32) * np.repeat(o[s], BLK, 1)[:, :cap, None])).to(dtype)
           for n, c, s in (("K", "k8", "ks"), ("V", "v8", "vs"))}

    def expect(got, tok):  # tok [BH, R]
        inside = (tok >= 0) & (tok < cap)
        at = tok.clamp(0, cap - 1)
        for g, n in zip(got, "KV"):
            want = torch.gather(ref[n], 1, at[..., None].expand(*at.shape, D)) * inside[..., None]
            assert g.dtype == dtype and torch.equal(g.cpu(), want)

    for pos, T in ((0, cap), (17, 1), (300, 64), (-5, 20), (1000, 3), (0, 0)):
        expect(st.read(pos, T, dtype), (pos + torch.arange(T))[None].expand(BH, T))
    pos = torch.tensor([0, 331, -2])
    expect(st.read(pos.to(DEV), 65, dtype), pos[:, None] + torch.arange(65))
    idx = torch.tensor([[5, 5, 332, 0, -1, 333, 64], [63, 64, 65, 2 ** 40, -(2 ** 40), 1, 2], [0] * 7])
    expect(st.gather_rows(idx.to(DEV), dtype), idx)
    expect(st.gather_rows(idx[:, :0].to(DEV), dtype), idx[:, :0])


# ----------------------------------------------------------------------------- attention
def _filled(BH, cap, D, code, lens, seed=10, spread=0.6):
    """A store whose rows hold lens tokens; what lies behind them is arbitrary, NaN among it."""
    st, o = _garbage(BH, cap, D, code, seed)
    for b, n in enumerate(lens):
        if n:
            K, V = _rand((1, n, D), seed + 2 * b, spread=spread), _rand((1, n, D), seed + 2 * b + 1, spread=spread)
            R.write_row(o["k8"][b], o["ks"][b], _f32(K)[0], 0, code)
            R.write_row(o["v8"][b], o["vs"][b], _f32(V)[0], 0, code)
    return _from_numpy(o, code), R.values(o["k8"], o["ks"], code), R.values(o["v8"], o["vs"], code)


def _close(got, b, g, want, bound):
    got = got[b, g].double().cpu().numpy()
    nan = np.isnan(want)  # NaN where, and only where, the formula has it
    assert np.array_equal(nan, np.isnan(got)), f"row {b} head {g}: NaN in other places"
    got, want, bound = got[~nan], want[~nan], bound[~nan]
    err = np.abs(got - want)
    assert (err <= bound).all(), f"row {b} head {g}: off by {(err / np.maximum(bound, 1e-300)).max():.3g} of its bound"


def _check(st, K, V, q, lens, length, window=0, softcap=None, slopes=None, idx=None, scale=None):
    qd = q.to(DEV)
    sl = None if slopes is None else slopes.to(DEV)
    if idx is None:
        got = st.attention(qd, length, window=window, scale=scale, softcap=softcap, slopes=sl)
    else:
        got = st.gather_attention(qd, idx.to(DEV), length, scale=scale, softcap=softcap, slopes=sl)
    assert got.dtype == torch.float32 and got.shape == q.shape
    sc = float(np.float32(q.shape[2] ** -0.5 if scale is None else scale))
    for b in range(q.shape[0]):
        n = max(0, min(int(lens[b]), st.cap))
        for g in range(q.shape[1]):
            toks = np.arange(max(0, n - window) if window else 0, n)
            if idx is not None:
                toks = idx[b, g].numpy()
                toks = toks[(toks >= 0) & (toks < n)]
            slope = None if slopes is None else float(slopes[b, g])
            want, bound = R.attention(q[b, g].double().numpy(), K[b], V[b], toks, n, sc, softcap or 0.0, slope)
            _close(got, b, g, want, bound)
    return got


def _q(BH, G, D, seed, dtype=torch.float32):
    return torch.randn(BH, G, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000])
def test_attention_lengths(code, D, n):
    st, K, V = _filled(2, 1003, D, code, [n, n])
    _check(st, K, V, _q(2, 4, D, n), [n, n], n)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 12, 16, 17])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention_heads_and_types(code, D, G, dtype):
    st, K, V = _filled(2, 640, D, code, [611, 611])
    _check(st, K, V, _q(2, G, D, G, dtype), [611, 611], 611)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 1, 63, 64, 65, 200, 5000])
@pytest.mark.parametrize("softcap, biased", [(None, False), (5.0, False), (None, True), (30.0, True)])
def test_attention_ragged(code, D, window, softcap, biased):
    """Rows of their own lengths, empty and out-of-range ones among them, with cap, bias and window."""
    lens = [0, 1, 64, 900, 1003, 65, 5000, -7]
    st, K, V = _filled(8, 1003, D, code, [min(max(n, 0), 1003) for n in lens])
    slopes = torch.rand(8, 3, generator=torch.Generator().manual_seed(1)) * 0.1 if biased else None
    for kind in (torch.int32, torch.int64):
        length = torch.tensor(lens, dtype=kind, device=DEV)
        got = _check(st, K, V, _q(8, 3, D, 5) * 2, lens, length, window, softcap, slopes)
        assert (got[0] == 0).all() and (got[7] == 0).all()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_long_row(code, D):
    lens = [20011, 7, 15000]
    st, K, V = _filled(3, 20020, D, code, lens)
    _check(st, K, V, _q(3, 4, D, 6), lens, torch.tensor(lens, dtype=torch.int32, device=DEV))
    _check(st, K, V, _q(3, 2, D, 6), [7] * 3, 7)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("k", [0, 1, 5, 31, 33, 128, 129, 512, 700, 2100])
def test_gather_attention(code, D, k):
    """Selections with tokens listed twice, padding, and tokens at or behind the row's end."""
    lens = [1000, 3, 0]
    st, K, V = _filled(3, 1003, D, code, lens)
    idx = torch.randint(-3, 1010, (3, 5, k), generator=torch.Generator().manual_seed(k))
    idx[0, 1] = -1                    # nothing selected
    idx[0, 2, : k // 2] = 17          # one token many times
    idx[0, 3] = torch.arange(k) % 1000
    if k > 2:
        idx[0, 4, :2] = torch.tensor([2 ** 40, -(2 ** 40)])
    length = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = _check(st, K, V, _q(3, 5, D, k), lens, length, idx=idx)
    assert (got[0, 1] == 0).all() and (got[2] == 0).all()
    slopes = torch.rand(3, 5, generator=torch.Generator().manual_seed(2)) * 0.05
    _check(st, K, V, _q(3, 5, D, k, torch.bfloat16) * 2, lens, length, softcap=8.0, slopes=slopes, idx=idx)
    _check(st, K, V, _q(3, 5, D, k, torch.float16), [3] * 3, 3, idx=idx, scale=0.3)


def test_gather_attention_whole_cap_by_default():
    st, K, V = _filled(1, 200, 128, "int8", [200])
    idx = torch.arange(200).view(1, 1, 200)
    _check(st, K, V, _q(1, 1, 128, 3), [200], None, idx=idx)


def test_selecting_every_token_is_dense_attention():
    st, K, V = _filled(2, 700, 128, "e4m3", [700, 700])
    q = _q(2, 3, 128, 8).to(DEV)
    idx = torch.randperm(700, generator=torch.Generator().manual_seed(3)).to(DEV).expand(2, 3, 700)
    a, b = st.attention(q, 700), st.gather_attention(q, idx)
    assert (a - b).abs().max() <= 1e-5 * a.abs().max()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_extreme_scores_and_values(code):
    """One score far above the rest, in the first or last token; scores all alike; large and small values and queries."""
    n, D = 1003, 128
    for hot in (0, 500, n - 1, None):
        o = {"k8": np.zeros((1, n, D), np.uint8), "v8": np.zeros((1, n, D), np.uint8),
             "ks": np.zeros((1, 16), np.float32), "vs": np.zeros((1, 16), np.float32)}
        K, V = _f32(_rand((1, n, D), 11))[0], _f32(_rand((1, n, D), 12))[0]
        V *= np.exp(np.linspace(-30, 20, n))[:, None].astype(np.float32)  # block scales over 20 decades
        q = _q(1, 2, D, 9)
        if hot is None:
            K[:] = K[0]
        else:
            K[hot] = 30.0 * q[0, 0].numpy()
        R.write_row(o["k8"][0], o["ks"][0], K, 0, code)
        R.write_row(o["v8"][0], o["vs"][0], V, 0, code)
        st = _from_numpy(o, code)
        Kv, Vv = R.values(o["k8"], o["ks"], code), R.values(o["v8"], o["vs"], code)
        for size, scale in ((1.0, None), (1e30, 1e-31), (1e-30, 1e29)):
            _check(st, Kv, Vv, (q * size), [n], n, scale=scale)
            _check(st, Kv, Vv, (q * size), [n], n, scale=scale, idx=torch.arange(n).expand(1, 2, n))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_negative_scales(code):
    """A negative score scale, and stores from elsewhere whose block scales have signs, or are 0."""
    st, K, V = _filled(2, 400, 64, code, [400, 390])
    for t, vals in ((st.k_scale, K), (st.v_scale, V)):
        t[:, 1::3] *= -1
        t[:, 4] = 0
        vals[:, np.arange(400) // BLK % 3 == 1] *= -1
        vals[:, 256:320] = 0
    q = _q(2, 3, 64, 4)
    idx = torch.randint(0, 390, (2, 3, 100), generator=torch.Generator().manual_seed(4))
    for scale, softcap in ((None, None), (-0.2, None), (-0.2, 4.0), (0.0, None)):
        _check(st, K, V, q, [390, 390], 390, softcap=softcap, scale=scale)
        _check(st, K, V, q, [390, 390], 390, softcap=softcap, scale=scale, idx=idx)


def test_nan_in_a_row_reaches_its_heads_only():
    st, K, V = _filled(2, 300, 128, "e4m3", [300, 300])
    st.v8.view(torch.uint8)[0, 150, 7] = 0x7F
    st.k8.view(torch.uint8)[1, 20, 3] = 0xFF
    q = _q(2, 2, 128, 4).to(DEV)
    for got in (st.attention(q, 300), st.gather_attention(q, torch.arange(300, device=DEV).expand(2, 2, 300))):
        assert got[0, :, 7].isnan().all() and got[0].isnan().sum() == 2 and got[1].isnan().all()
    assert not st.attention(q, 150)[0].isnan().any() and not st.attention(q, 300, window=149)[0].isnan().any()
    q[0, 0, 0] = float("nan")
    got = st.attention(q, 140)
    assert got[0, 0].isnan().all() and not got[0, 1].isnan().any()


def test_refusals():
    st = RowStore8.empty(2, 100, torch.int8, 64, DEV)
    K = torch.zeros(2, 10, 64, device=DEV)
    q, idx = torch.zeros(2, 3, 64, device=DEV), torch.zeros(2, 3, 5, dtype=torch.int64, device=DEV)
    for bad in (lambda: st.write(K, K, 2 ** 64), lambda: st.attention(q, 2 ** 64 + 5), lambda: st.read(2 ** 64, 5),
                lambda: st.write(K, K, 91), lambda: st.write(K, K, -1), lambda: st.write(K, K[:, :5]), lambda: st.write(K, K.half()),
                lambda: st.write(K[:1], K[:1]), lambda: st.write(K[..., :32], K[..., :32]), lambda: st.write(K.cpu(), K),
                lambda: st.write(K, K, torch.zeros(3, dtype=torch.int32, device=DEV)),
                lambda: st.write(K, K, torch.zeros(2, device=DEV)), lambda: st.read(0, 5, torch.int32), lambda: st.read(0, -1),
                lambda: st.gather_rows(idx), lambda: st.attention(q, 101), lambda: st.attention(q, -1),
                lambda: st.attention(q, 5, window=-1), lambda: st.attention(q[:, :0], 5), lambda: st.attention(q[0], 5),
                lambda: st.attention(q, 5, softcap=-2.0), lambda: st.attention(q, torch.tensor([5, 5])),
                lambda: st.gather_attention(q, idx[:, :2]), lambda: st.gather_attention(q, idx, 101),
                lambda: st.gather_attention(q, idx.cpu()),
                lambda: RowStore8(st.k8, st.v8[:, :50], st.k_scale, st.v_scale),
                lambda: RowStore8(st.k8, st.v8, st.k_scale[:, :1], st.v_scale),
                lambda: RowStore8(st.k8.float(), st.v8.float(), st.k_scale, st.v_scale),
                lambda: RowStore8(st.k8[:, ::2], st.v8[:, ::2], st.k_scale[:, :1], st.v_scale[:, :1]),
                lambda: RowStore8.empty(2, 100, torch.int8, 96, DEV)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


# ----------------------------------------------------------------------------- together
def test_decode_with_the_key_index():
    """A prompt into the key index and the row store, then steps: write the token, select with the index, attend over the
    selection, and over everything."""
    BH, n, G, k = 2, 2000, 4, 256
    K, V = _rand((BH, n, 128), 20, torch.bfloat16, 0.5), _rand((BH, n, 128), 21, torch.bfloat16, 0.5)
    st, o = _empty(BH, n + 10, 128, "e4m3")
    st.write(K.to(DEV), V.to(DEV))
    R.write(o, _f32(K), _f32(V), 0, "e4m3")
    index = bp.PlaneStore(K.to(DEV))
    var = K[:, 16:].float().var(1).to(DEV)
    for step in range(3):
        at = n + step
        kt, vt = _rand((BH, 1, 128), 30 + step, torch.bfloat16), _rand((BH, 1, 128), 40 + step, torch.bfloat16)
        st.write(kt.to(DEV), vt.to(DEV), at)
        R.write(o, _f32(kt), _f32(vt), at, "e4m3")
        q = _q(BH, G, 128, 50 + step)
        qd = q.to(DEV)
        g = ((qd ** 2) * var[:, None]).sum(1)
        idx = index.plan_scan_topk(qd, g, 48.0, k)
        new = torch.arange(n, at + 1, device=DEV).expand(BH, G, step + 1)
        idx = torch.cat([idx, new], 2)
        _same(st, o, "e4m3")
        Kv, Vv = R.values(o["k8"], o["ks"], "e4m3"), R.values(o["v8"], o["vs"], "e4m3")
        _check(st, Kv, Vv, q, [at + 1] * BH, at + 1, idx=idx.cpu())
        _check(st, Kv, Vv, q, [at + 1] * BH, at + 1)


def test_captured_step_replayed():
    """A step in a graph (write, dense and selected attention, read back) over growing rows: every replay equals the same
    calls made eagerly, with eager work between the replays."""
    BH, cap, G, D = 4, 700, 5, 128
    st = RowStore8.empty(BH, cap, torch.int8, D, DEV)
    eager = RowStore8.empty(BH, cap, torch.int8, D, DEV)
    K, V = _rand((BH, 600, D), 60, torch.bfloat16).to(DEV), _rand((BH, 600, D), 61, torch.bfloat16).to(DEV)
    for s in (st, eager):
        s.write(K, V)
    pos = torch.tensor([600, 599, 63, 10], dtype=torch.int32, device=DEV)
    length = pos + 1
    kt, vt = torch.zeros(BH, 1, D, device=DEV), torch.zeros(BH, 1, D, device=DEV)
    q = torch.zeros(BH, G, D, device=DEV)
    idx = torch.zeros(BH, G, 40, dtype=torch.int64, device=DEV)

    def step(s):
        s.write(kt, vt, pos)
        return s.attention(q, length), s.gather_attention(q, idx, length), *s.read(pos, 1, torch.float32)

    step(eager)  # the first calls load the kernels
    step(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(st)
    gen = torch.Generator(device=DEV).manual_seed(3)
    for i in range(6):
        kt.normal_(generator=gen).mul_(1 + i)
        vt.normal_(generator=gen)
        q.normal_(generator=gen)
        idx.random_(-1, 600, generator=gen)
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        assert torch.equal(st.k8, eager.k8) and torch.equal(st.k_scale, eager.k_scale)
        pos += 1
        length += 1


def test_two_streams_at_once():
    """Two stores' calls on two streams at once, and one store's attention on both, equal the same calls one by one."""
    stores = [_filled(4, 5000, 128, c, [5000] * 4)[0] for c in ("e4m3", "int8")]
    q = _q(4, 4, 128, 1).to(DEV)
    idx = torch.randint(0, 5000, (4, 4, 512), generator=torch.Generator().manual_seed(1)).to(DEV)
    want = [(s.attention(q, 5000), s.gather_attention(q, idx)) for s in stores]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            s = stores[(i // 2) % 2]
            got.append((s.attention(q, 5000), s.gather_attention(q, idx)))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        for a, b in zip(pair, want[(i // 2) % 2]):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows behind the first 4 GiB of codes."""
    BH, cap, D = 3, 17_000_000, 128
    st = RowStore8.empty(BH, cap, torch.int8, D, DEV)
    n, T = cap - 3, 130
    K, V = _rand((BH, T, D), 70), _rand((BH, T, D), 71)
    st.write(K.to(DEV), V.to(DEV), n - T)
    got = st.read(n - T, T, torch.float32)
    p = (n - T) % BLK
    o = {"k8": np.zeros((BH, T + p, D), np.uint8), "v8": np.zeros((BH, T + p, D), np.uint8),
         "ks": np.zeros((BH, 4), np.float32), "vs": np.zeros((BH, 4), np.float32)}
    R.write(o, _f32(K), _f32(V), p, "int8")
    Kv, Vv = R.values(o["k8"], o["ks"], "int8"), R.values(o["v8"], o["vs"], "int8")
    assert np.array_equal(got[0].cpu().numpy(), Kv[:, p:].astype(np.float32))
    assert np.array_equal(got[1].cpu().numpy(), Vv[:, p:].astype(np.float32))
    q = _q(BH, 2, D, 72)
    out = st.attention(q.to(DEV), n, window=100)
    idx = torch.arange(n - 100, n).expand(BH, 2, 100).to(DEV)
    sel = st.gather_attention(q.to(DEV), idx, n)
    for b in range(BH):
        for g in range(2):
            want, bound = R.attention(q[b, g].double().numpy(), Kv[b], Vv[b], np.arange(T + p - 100, T + p), T + p,
                                      float(np.float32(D ** -0.5)))
            _close(out, b, g, want, bound)
            _close(sel, b, g, want, bound)


# ----------------------------------------------------------------------------- how rows are shared out
@pytest.mark.parametrize("BH, cap", [(70, 3000), (200, 1500), (300, 1200), (600, 1200)])
@pytest.mark.parametrize("G", [2, 20])
def test_attention_many_rows(BH, cap, G):
    """More rows than one wave has lanes, and more than the workgroups of a call; rows without tokens among them."""
    rng = np.random.default_rng(BH)
    lens = rng.integers(0, cap + 1, BH)
    lens[[0, BH // 2, BH - 1]] = [0, cap, 0]
    lens[rng.integers(0, BH, 5)] = 1
    st, K, V = _filled(BH, cap, 64, "int8", lens)
    q = _q(BH, G, 64, 7)
    got = st.attention(q.to(DEV), torch.from_numpy(lens.astype(np.int32)).to(DEV))
    some = sorted({0, 1, 63, BH - 1, BH // 2, *rng.integers(0, BH, 12).tolist()})
    for b in some:
        for g in (0, G - 1):
            want, bound = R.attention(q[b, g].double().numpy(), K[b], V[b], np.arange(lens[b]), lens[b],
                                      float(np.float32(64 ** -0.5)))
            _close(got, b, g, want, bound)
    listed = torch.arange(cap).expand(BH, G, cap).contiguous().to(DEV)
    every = st.gather_attention(q.to(DEV), listed, torch.from_numpy(lens.astype(np.int32)).to(DEV))
    assert (got - every).abs().max() <= 2e-5 * every.abs().max()


@pytest.mark.parametrize("BH, G", [(520, 2), (65, 9)])
def test_one_long_row_among_many(BH, G):
    """A batch of short rows with a few long ones: every row equals the call on that row alone."""
    cap, D = 9000, 64
    st = RowStore8.empty(BH, cap, torch.float8_e4m3fn, D, DEV)
    gen = torch.Generator(device=DEV).manual_seed(BH)
    for t in (st.k8, st.v8):
        t.view(torch.uint8).random_(0, 96, generator=gen).bitwise_xor_((torch.rand(t.shape, generator=gen, device=DEV) < 0.5) * 128)
    for t in (st.k_scale, st.v_scale):
        t.uniform_(0.1, 1.0, generator=gen)
    lens = torch.randint(0, 200, (BH,), generator=gen, device=DEV, dtype=torch.int32)
    lens[[3, BH // 2, BH - 1]] = torch.tensor([9000, 8001, 4000], dtype=torch.int32, device=DEV)
    q = torch.randn(BH, G, D, generator=gen, device=DEV)
    got = st.attention(q, lens)
    for b in (0, 1, 2, 3, 4, 63, 64, BH // 2, BH - 2, BH - 1):
        alone = RowStore8(st.k8[b:b + 1], st.v8[b:b + 1], st.k_scale[b:b + 1], st.v_scale[b:b + 1])
        want = alone.attention(q[b:b + 1], int(lens[b]))
        assert (got[b] - want[0]).abs().max() <= 2e-5 * want.abs().max(), b


@pytest.mark.parametrize("BH, G, D", [(1, 1, 128), (3, 5, 64), (2, 33, 128)])
def test_attention_every_share(BH, G, D):
    """Lengths and windows across every way of sharing a row out: one length, one length as a tensor, and the list of the
    same tokens agree."""
    cap = 40000
    st, _, _ = _filled(BH, cap, D, "e4m3", [cap] * BH, spread=0.3)
    q = _q(BH, G, D, 3).to(DEV)
    ns = [1, 60, 64, 65, 200, 256, 257, 320, 500, 512, 513, 1023, 1024, 1025, 1087, 1088, 1089, 1100, 2047, 2049, 4095, 4160, 8191,
          8200, 16383, 16385, 20000, 32767, 39999, 40000]
    for i, n in enumerate(ns):
        for window in (0, ns[(i * 7) % len(ns)]):
            lo = max(0, n - window) if window else 0
            a = st.attention(q, n, window=window)
            b = st.attention(q, torch.full((BH,), n, dtype=torch.int32, device=DEV), window=window)
            c = st.gather_attention(q, torch.arange(lo, n, device=DEV).expand(BH, G, n - lo))
            size = c.abs().max()
            assert (a - c).abs().max() <= 2e-5 * size and (b - c).abs().max() <= 2e-5 * size, (n, window)


@pytest.mark.parametrize("window", [1, 64, 1000, 1090, 4096, 19999])
def test_attention_long_windows(window):
    lens = [20011, 7, 15000, 0, 4097]
    st, K, V = _filled(5, 20020, 64, "int8", lens)
    slopes = torch.rand(5, 3, generator=torch.Generator().manual_seed(4)) * 0.01
    _check(st, K, V, _q(5, 3, 64, 6), lens, torch.tensor(lens, dtype=torch.int32, device=DEV), window, 20.0, slopes)


def test_captured_long_rows_replayed():
    """Rows shared out by lengths on the device, in a graph whose lengths grow between replays."""
    BH, cap, G, D = 3, 30000, 4, 128
    st, _, _ = _filled(BH, cap, D, "e4m3", [cap] * BH, spread=0.3)
    q, length = torch.zeros(BH, G, D, device=DEV), torch.tensor([100, 0, 29000], dtype=torch.int32, device=DEV)
    q.normal_()
    st.attention(q, length)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same store, replayed in turn and together
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((st.attention(q, length), st.attention(q, length, window=5000)))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        q.normal_()
        want = st.attention(q, length), st.attention(q, length, window=5000)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for pair in outs:
            assert all(torch.equal(a, b) for a, b in zip(pair, want))
        length.copy_((length * 2 + 77) % (cap + 1))


def test_query_layouts():
    """Queries with any strides and addresses, of other types, and slopes per head."""
    st, K, V = _filled(2, 500, 64, "int8", [500, 500])
    wide = torch.randn(2, 3, 200, generator=torch.Generator().manual_seed(5)).to(DEV)
    slopes = torch.tensor([0.1, 0.2, 0.05], device=DEV)
    idx = torch.arange(500, device=DEV).expand(2, 3, 500)
    for q in (wide[..., 3:67], wide[..., :64].transpose(0, 1).contiguous().transpose(0, 1), wide[..., :64].double()):
        same = q.float().contiguous()
        every = slopes.expand(2, 3).contiguous()
        assert torch.equal(st.attention(q, 500, slopes=slopes), st.attention(same, 500, slopes=every))
        assert torch.equal(st.gather_attention(q, idx.int(), 500, slopes=slopes.double()),
                           st.gather_attention(same, idx.contiguous(), 500, slopes=every))


def test_same_result_twice():
    st, _, _ = _filled(4, 9000, 128, "e4m3", [9000, 1, 5000, 8999])
    q = _q(4, 9, 128, 2).to(DEV)
    lens = torch.tensor([9000, 1, 5000, 8999], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, 9000, (4, 9, 700), generator=torch.Generator().manual_seed(2)).to(DEV)
    for call in (lambda: st.attention(q, lens), lambda: st.attention(q, 8000), lambda: st.gather_attention(q, idx, lens)):
        first = call().view(torch.int32)  # bits: rows past their written tokens hold NaN
        assert all(torch.equal(first, call().view(torch.int32)) for _ in range(5))
