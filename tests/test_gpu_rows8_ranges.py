"""The 8-bit K/V row store at the ends of its ranges: large scores, scales and queries of very different sizes, extreme caps,
many heads with cap and bias."""
import numpy as np
import pytest
import torch

from fathom_amd import _lib
from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R
from test_gpu_rows8 import BLK, DEV, _check, _close, _f32, _filled, _from_numpy, _q, _rand, _same

pytestmark = pytest.mark.gpu


def _rows(K, V, code):
    """A store of the rows K, V [BH, n, D], and its values."""
    BH, n, D = K.shape
    nblk = -(-n // BLK)
    o = {"k8": np.zeros((BH, n, D), np.uint8), "v8": np.zeros((BH, n, D), np.uint8),
         "ks": np.zeros((BH, nblk), np.float32), "vs": np.zeros((BH, nblk), np.float32)}
    R.write(o, np.asarray(K, np.float32), np.asarray(V, np.float32), 0, code)
    return _from_numpy(o, code), R.values(o["k8"], o["ks"], code), R.values(o["v8"], o["vs"], code)


# ----------------------------------------------------------------------------- large scores
def _both(st, q, n, lens=None, **kw):
    """Dense attention, and attention over the list of the same tokens."""
    BH, G, _ = q.shape
    idx = torch.arange(n, device=DEV).expand(BH, G, n)
    return st.attention(q, n if lens is None else lens, **kw), st.gather_attention(q, idx, n, **kw)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("score", [1e5, 3e6, 1e8, -1e8, 1e10, -1e10, 1e20, -1e20])
def test_large_scores(code, D, score):
    """Scores far past 2^24.  Tokens of equal keys have equal weights, whatever their score: the mean of V.  One token
    whose score is that far above the rest: its V.  The weights are exact then, so that what is left are the sums
    (2^-24 for each token, as in the oracle's bound) and a weight's two f16 parts."""
    for n in (1, 2, 65, 300, 1500, 5000):
        rng = np.random.default_rng(n)
        G = 3
        k0, V = rng.standard_normal((1, 1, D)), rng.standard_normal((1, n, D))
        st, K, v = _rows(np.repeat(k0, n, 1), V, code)
        q = _q(1, G, D, 3).double()
        q *= score * D ** 0.5 / (q @ torch.from_numpy(K[0, 0]))[..., None]
        q = q.float().to(DEV)
        size = (n / 8 + 64) * R.U + 2.0 ** -20
        for slopes in (None, torch.zeros(1, G, device=DEV)):
            for got in _both(st, q, n, slopes=slopes):
                err = np.abs(got[0].double().cpu().numpy() - v[0].mean(0))
                assert (err <= size * np.abs(v[0]).mean(0) + n * 2.0 ** -37 * np.abs(v).max()).all(), (n, err.max())
        for hot in {0, n // 2, n - 1}:  # the others' keys are zero, or the hot one's where scores are negative
            K1 = np.zeros((1, n, D)) if score > 0 else np.repeat(k0, n, 1)
            K1[0, hot] = k0[0, 0] if score > 0 else 0.0
            st, K, v = _rows(K1, V, code)
            for slopes in (None, torch.zeros(1, G, device=DEV)):
                for got in _both(st, q, n, slopes=slopes):
                    err = np.abs(got[0].double().cpu().numpy() - v[0, hot])
                    assert (err <= size * np.abs(v[0, hot])).all(), (n, hot, err.max())


def test_scores_that_differ_by_little_beside_their_size():
    """Scores near 2^21 whose differences float32 still holds: weights go by the differences."""
    n, D, G = 200, 64, 2
    K, V = np.zeros((1, n, D)), np.random.default_rng(1).standard_normal((1, n, D))
    K[0, :, 0] = 127 / 64  # the block's scale is 1 / 64, and every key a code
    K[0, :, 1] = np.array([0, 64, 127])[np.arange(n) % 3] / 64
    st, Kv, v = _rows(K, V, "int8")
    assert np.array_equal(Kv, K)
    q = torch.zeros(1, G, D)
    q[0, :, 0], q[0, :, 1] = 2.0 ** 20, 8.0
    z = Kv[0] @ q[0, 0].double().numpy()
    # Two products, two sums (or one, and the factor) and the factor's product round a score here, each by 2^-24 of it, at
    # most two half steps: compare with the weights that scores moved by eight half steps can have.
    step = 8 * 2.0 ** (np.floor(np.log2(np.abs(z).max())) - 24)
    w = np.exp(z - z.max())
    lo, hi = w * np.exp(-step), w * np.exp(step)
    lo, hi = lo / hi.sum(), hi / lo.sum()
    a, b = lo[:, None] * v[0], hi[:, None] * v[0]
    least, most = np.minimum(a, b).sum(0), np.maximum(a, b).sum(0)
    slack = 2.0 ** -18 * (hi @ np.abs(v[0]))
    for got in _both(st, q.to(DEV), n, scale=1.0):
        got = got[0].double().cpu().numpy()
        assert (got >= least - slack).all() and (got <= most + slack).all()


# ----------------------------------------------------------------------------- scales of V far apart
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D, G", [(64, 3), (128, 3), (64, 12), (128, 12)])
@pytest.mark.parametrize("power", [20, 40, 60])
def test_large_values_without_weight(code, D, G, power):
    """Blocks of large values whose tokens have next to no weight, before, behind and among those that have it: the others'
    values keep their bits."""
    for n, where in ((500, "first"), (500, "last"), (1000, "first"), (1000, "every fifth"), (4000, "first"), (4000, "last")):
        rng = np.random.default_rng(power)
        K, V = rng.standard_normal((1, n, D)), rng.standard_normal((1, n, D))
        blk = np.arange(n) // BLK
        big = blk == 0 if where == "first" else blk == blk[-1] if where == "last" else blk % 5 == 0
        V[0, big] *= 2.0 ** power
        q = _q(1, G, D, 5)
        far = -(power * np.log(2.0) + 30.0) * D ** 0.5  # the large values' weights: e^-30 beside their size
        K[0, :, 0] = np.where(big, far / 8, 0.0)
        q[..., 0] = 8.0
        st, Kv, Vv = _rows(K, V, code)
        _check(st, Kv, Vv, q, [n], n)
        _check(st, Kv, Vv, q, [n], torch.tensor([n], dtype=torch.int32, device=DEV))
        _check(st, Kv, Vv, q, [n], n, softcap=1e4, slopes=torch.full((1, G), 1e-3))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("falls", [True, False])
def test_values_and_weights_over_many_decades(code, falls):
    """Scales of V and weights that rise and fall together or against each other, over more than the float32 range."""
    n, D = 1500, 64
    rng = np.random.default_rng(2)
    t = np.linspace(1.0, 0.0, n) if falls else np.linspace(0.0, 1.0, n)
    for values, weights in ((60, 0), (60, 40), (60, -40), (-60, 200), (60, -200)):
        K, V = np.zeros((1, n, D)), rng.standard_normal((1, n, D)) * np.exp(values * t)[:, None]
        K[0, :, 0] = weights * t
        q = torch.zeros(1, 2, D)
        q[0, :, 0] = 1.0
        st, Kv, Vv = _rows(K, V, code)
        _check(st, Kv, Vv, q, [n], n, scale=1.0)


# ----------------------------------------------------------------------------- queries
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D, G", [(64, 3), (128, 3), (64, 12), (128, 12)])
@pytest.mark.parametrize("power", [12, 20, 30, 45])
def test_queries_with_a_large_channel(code, D, G, power):
    """A query channel far above the others whose keys are zero: the scores come from the others."""
    for n in (100, 1500):
        rng = np.random.default_rng(power)
        K, V = rng.standard_normal((1, n, D)), rng.standard_normal((1, n, D))
        K[..., [5, 40]] = 0.0
        st, Kv, Vv = _rows(K, V, code)
        q = _q(1, G, D, power) * 2.0
        q[..., 5] = 2.0 ** power
        q[0, 1, 40] = -(2.0 ** power)
        _check(st, Kv, Vv, q, [n], n)
        _check(st, Kv, Vv, q, [n], n, softcap=20.0, slopes=torch.full((1, G), 0.01))
        _check(st, Kv, Vv, q, [n], n, idx=torch.arange(n).expand(1, G, n))
    q[0, 0] = 0.0
    _check(st, Kv, Vv, q, [n], n)


# ----------------------------------------------------------------------------- arguments
def test_negative_windows_are_refused():
    n, D = 300, 64
    st, _, _ = _filled(1, n, D, "int8", [n])
    q = _q(1, 2, D, 6).to(DEV)
    for window in (-1, -(2 ** 63), -(2 ** 64), -(2 ** 64) + 5):  # the last two wrap to 0 and 5
        with pytest.raises(ValueError):
            st.attention(q, n, window=window)


def test_lengths_of_every_integer_type():
    n, D = 300, 64
    st, K, V = _filled(3, n, D, "int8", [n] * 3)
    q = _q(3, 2, D, 6)
    for dtype, lens in ((torch.uint64, [5, 2 ** 63, 2 ** 32]), (torch.uint32, [5, 2 ** 32 - 1, 2 ** 31]),
                        (torch.int64, [5, 2 ** 62, 2 ** 32]), (torch.uint16, [5, 65535, 300]), (torch.int16, [-1, 299, 0]),
                        (torch.uint8, [5, 255, 100]), (torch.int8, [127, -128, 1])):
        _check(st, K, V, q, lens, torch.tensor(lens, dtype=dtype, device=DEV))


def test_read_far_behind_the_store():
    """Places at the ends of 64 bits are outside the store: zero rows, from the C call too."""
    st, _, _ = _filled(2, 100, 64, "int8", [100, 100])
    K, V = torch.ones(2, 2, 7, 64, device=DEV)
    for at in (2 ** 63 - 1, 2 ** 63 - 4, -(2 ** 63), -(2 ** 63) + 5, 100, -7):
        K.fill_(1.0)
        V.fill_(1.0)
        _lib.call("fathom_rows8_read", st.k8.data_ptr(), st.v8.data_ptr(), st.k_scale.data_ptr(), st.v_scale.data_ptr(),
                  _lib.DT_I8, 2, 100, 64, None, None, at, 7, _lib.DT_F32, K.data_ptr(), V.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        assert not K.any() and not V.any(), at
    full = st.read(0, 100, torch.float32)[0]
    assert torch.equal(st.read(-3, 7, torch.float32)[0][:, 3:], full[:, :4])


def test_more_heads_than_one_axis_of_a_grid_takes():
    """BH G past 2^24, at lengths of their own: splits and their join."""
    BH, G, D, cap = 65535, 257, 64, 1100
    st = RowStore8.empty(BH, cap, torch.int8, D, DEV)
    st.v8[:, :3] = (torch.arange(3 * D, device=DEV) - 96).to(torch.int8).view(3, D)
    st.v_scale.fill_(0.5)
    rows = [0, 1, 300, 40000, BH - 1]
    lens = torch.zeros(BH, dtype=torch.int32, device=DEV)
    for i, b in enumerate(rows):
        lens[b] = i % 3 + 1
    lens[300] = cap
    q = torch.zeros(BH, G, D, dtype=torch.float16, device=DEV)  # every score 0: means of V
    got = st.attention(q, lens)
    for b in rows:
        n = int(lens[b])
        want = st.v8[b, :n].double().mul(0.5).mean(0)
        assert (got[b].double() - want).abs().max() <= 2.0 ** -20 * want.abs().max(), b
    got[rows] = 0
    assert not got.any()


# ----------------------------------------------------------------------------- caps
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e-10, 1.0, 1e10])
def test_extreme_caps(code, D, size):
    """A cap far below the scores leaves every token the same weight; one far above them changes nothing."""
    for softcap in (1e-300, 1e-50, 1e-38, 1e-20, 1e-4, 1e10, 1e20, 1e26, 1e28, 1e32, 1e38, 1e200):
        if size > 1.0 and softcap > 1e4:
            size = 30.0  # scores of 1e10 differ by more than a float32 bound can say
        n = 300
        st, K, V = _filled(1, n, D, code, [n])
        K = K.copy()
        st.k_scale[0, 2], K[0, 128:192] = 0.0, 0.0
        st.k8.view(torch.uint8)[0, 70], K[0, 70] = 0, 0.0
        q = _q(1, 2, D, 4) * size
        for idx in (None, torch.arange(n).expand(1, 2, n)):
            with np.errstate(over="ignore"):
                got = _check(st, K, V, q, [n], n, softcap=softcap, idx=idx)
            if softcap <= 1e-4:  # scores within the cap: weights within e^(2 cap) of each other
                err = np.abs(got[0].double().cpu().numpy() - V[0].mean(0))
                assert (err <= (2.1 * softcap + (n / 8 + 64) * R.U + 2.0 ** -20) * np.abs(V[0]).mean(0)).all()


# ----------------------------------------------------------------------------- cap and bias with many heads
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [9, 12, 16, 17, 25])
def test_cap_and_bias_of_many_heads(code, D, G):
    """More than eight heads, with slopes of their own: rows of one workgroup and split ones, of one length and of their
    own, with and without a window."""
    slopes = torch.exp2(-torch.linspace(2.0, 9.0, 2 * G)).view(2, G).flip(1)
    q = _q(2, G, D, G) * torch.linspace(0.5, 4.0, G)[None, :, None]
    for cap, lens, window in ((700, [650, 333], 0), (2500, [2490, 1300], 0), (2500, [2490, 70], 1500), (130, [100, 1], 0)):
        st, K, V = _filled(2, cap, D, code, lens)
        for softcap, bias in ((5.0, None), (None, slopes), (30.0, slopes)):
            _check(st, K, V, q, lens, torch.tensor(lens, dtype=torch.int32, device=DEV), window, softcap, bias)
            _check(st, K, V, q, [min(lens)] * 2, min(lens), window, softcap, bias)


# ----------------------------------------------------------------------------- writes
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_write_into_blocks_of_signed_and_zero_scales(code):
    """Stores from elsewhere: a block keeps its scale's sign, and values of a scale of 0 stay 0."""
    D, n = 64, 40
    rng = np.random.default_rng(3)
    o = {x: rng.integers(0, 127, (4, 64, D), dtype=np.uint8) for x in ("k8", "v8")}
    o["ks"] = np.array([[-0.02], [0.0], [-1e-4], [-0.0]], np.float32)
    o["vs"] = np.array([[0.0], [-0.5], [0.01], [-3.0]], np.float32)
    st = _from_numpy(o, code)
    before = st.read(0, n, torch.float32)
    K, V = _rand((4, 3, D), 8), _rand((4, 3, D), 9)
    st.write(K.to(DEV), V.to(DEV), n)
    R.write(o, _f32(K), _f32(V), n, code)
    _same(st, o, code)
    for got, was, new in zip(st.read(0, n + 3, torch.float32), before, (K, V)):
        # half a step of a scale that grew, at most twice largest / 448 or 127 (e4m3: or of the value), or of the earlier one
        new = new.to(DEV)
        step = new.abs().amax((1, 2)) * (2.0 ** -4 if code == "e4m3" else 1.0 / 127) + was.abs().amax((1, 2)) * 2.0 ** -7
        assert ((got[:, :n] - was).abs() <= step[:, None, None]).all()
        assert ((got[:, n:] - new).abs() <= step[:, None, None]).all()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_scales_that_are_not_finite(code, bad):
    """A block of such a scale of K makes NaN of the heads of its row, of V the channels' values (NaN for a code of 0 or beside
    other signs); rows that do not hold it are as before, and so is a call that ends before it."""
    st, K, V = _filled(3, 300, 64, code, [300] * 3)
    q = _q(3, 2, 64, 3)
    st.k_scale[0, 2] = bad
    st.v_scale[1, 2] = bad
    for softcap in (None, 5.0):
        for idx in (None, torch.arange(300).expand(3, 2, 300)):
            got = (st.attention(q.to(DEV), 300, softcap=softcap) if idx is None
                   else st.gather_attention(q.to(DEV), idx.to(DEV), 300, softcap=softcap))
            assert not got[1].isfinite().any()
            if softcap is None or bad != bad:
                assert got[0].isnan().all()
            for g in (0, 1):
                want = R.attention(q[2, g].double().numpy(), K[2], V[2], np.arange(300), 300, 64 ** -0.5, softcap or 0.0)
                _close(got, 2, g, *want)
    _check(st, K, V, q, [128] * 3, 128)
