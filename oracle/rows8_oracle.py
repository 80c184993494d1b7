"""numpy restatement of the 8-bit K/V row store: the writer bit for bit, reading,
and attention in float64.  Test infrastructure only.

A store is a dict of bytes k8, v8 [BH, cap, D] (uint8; int8 codes as their two's
complement bytes) and float32 scales ks, vs [BH, ceil(cap / 64)]."""
import numpy as np

BLK = 64
MIN_SCALE = np.float32(2.0 ** -100)
U = 2.0 ** -24  # half a step of float32


def _e4m3_table():
    """The 128 non-negative values: e = 0 subnormals, 0x7F NaN."""
    v = np.empty(128)
    for c in range(128):
        e, m = c >> 3, c & 7
        v[c] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
    v[127] = np.nan
    return v


E4M3 = _e4m3_table()


def qmax(code):
    return 127.0 if code == "int8" else 448.0


def decode(b, code):
    b = np.asarray(b, np.uint8)
    if code == "int8":
        return b.view(np.int8).astype(np.float64)
    return np.where(b & 0x80, -1.0, 1.0) * E4M3[b & 0x7F]


def encode(y, code):
    """Nearest code, ties to the even code; infinities saturate."""
    y = np.asarray(y, np.float64)
    if code == "int8":
        v = np.rint(np.clip(np.where(np.isnan(y), 0.0, y), -127, 127))
        return v.astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(np.where(np.isnan(y), 0.0, y)), 448.0)
    hi = np.searchsorted(E4M3[:127], a)  # the first value >= a
    lo = np.maximum(hi - 1, 0)
    up, down = E4M3[hi] - a, a - E4M3[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    c = np.where(np.isnan(y), 0x7F, c).astype(np.uint8)
    return c | (np.signbit(y).astype(np.uint8) << 7)


def grown(was, need):
    """The least was * 2^j, j >= 0, that reaches need, and j."""
    j = 0
    while np.float64(was) * 2.0 ** j < np.float64(need):
        j += 1
    return np.float32(np.float64(was) * 2.0 ** j), j


def write_row(codes, scale, x, p, code):
    """Rows x [T, D] (their values as float32) into codes [cap, D] and scale at p."""
    T = x.shape[0]
    if T == 0 or p < 0 or p + T > codes.shape[0]:
        return
    x = np.asarray(x, np.float32)
    for b in range(p // BLK, (p + T - 1) // BLK + 1):
        lo, hi = max(p, b * BLK), min(p + T, (b + 1) * BLK)
        new = x[lo - p:hi - p]
        a = np.abs(new)[np.isfinite(new)]
        with np.errstate(over="ignore"):
            need = np.maximum((a.max() if a.size else np.float32(0)) / np.float32(qmax(code)), MIN_SCALE)
        was = scale[b]
        s = need
        if p > b * BLK and np.isfinite(was):
            j = None  # earlier values are 0
            if was:
                s, j = grown(abs(was), need)
                s = np.copysign(s, was)
            if j != 0:
                old = decode(codes[b * BLK:p], code).astype(np.float32) * np.float32(2.0 ** -j if j else 0.0)
                codes[b * BLK:p] = encode(old, code)
        with np.errstate(over="ignore", invalid="ignore"):
            codes[lo:hi] = encode(new * (np.float32(1.0) / s), code)
        scale[b] = s


def write(store, K, V, pos, code):
    for b in range(K.shape[0]):
        p = int(pos[b]) if np.ndim(pos) else int(pos)
        write_row(store["k8"][b], store["ks"][b], K[b], p, code)
        write_row(store["v8"][b], store["vs"][b], V[b], p, code)


def values(codes, scale, code):
    """float64 values [..., cap, D] of codes and scales."""
    s = np.repeat(np.asarray(scale, np.float64), BLK, -1)[..., :codes.shape[-2]]
    return decode(codes, code) * s[..., None]


def attention(q, K, V, toks, length, scale, softcap=0.0, slope=None):
    """One query head in float64 over values K, V [cap, D] and tokens toks.  Returns
    (out [D], the bound of a float32 evaluation's error [D]).

    The bound: a score is a sum of D products, each product and partial sum off by at
    most U relative to the sum of their sizes (A), the scale, cap and bias a few more U of the
    score's size; a score's error enters its weight e^z, once above and once below the
    fraction.  Sums over tokens run in chains of at most an eighth of them plus the
    joins; a weight w held as two f16 parts is off by 2^-22 of itself, or by 2^-38 of the
    largest w s of a token (s: its block's scale of V) times the format's largest code, which is at most
    twice the largest |V| of the block."""
    D = q.shape[0]
    if len(toks) == 0:
        return np.zeros(D), np.zeros(D)
    k, v = K[toks], V[toks]
    u = k @ q * scale
    a = (np.abs(k) @ np.abs(q)).max() * abs(scale)
    z = softcap * np.tanh(u / softcap) if softcap else u
    bias = slope * (np.asarray(toks, np.float64) - (length - 1)) if slope is not None else np.zeros(len(toks))
    z = z + bias
    m = z.max()
    p = np.exp(z - m)
    w = p / p.sum()
    weight = w @ np.abs(v)
    dz = (D + 24) * U * a + 8 * U * (np.abs(z).max() + np.abs(bias).max())
    rel = 2 * dz + (len(toks) / 8 + 64) * U + 2.0 ** -20
    blocks = np.nan_to_num(np.abs(np.pad(V, ((0, -len(V) % BLK), (0, 0))))).reshape(-1, BLK * D).max(1)
    return w @ v, rel * weight + len(toks) * 2.0 ** -37 * (w * blocks[np.asarray(toks) // BLK]).max()
