"""The 8-bit K/V row store at the ends of its ranges: large scores, scales and queries of very different sizes, extreme caps,
many heads with cap and bias."""
import numpy as np
import pytest
import torch

from fathom_amd import _lib
from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R
from test_gpu_rows8 import BLK, DEV, _check, _close, _f32, _filled, _from_numpy, _q, _rand

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
