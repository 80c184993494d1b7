"""Rotated writes into the 8-bit K/V row store on the GPU: bit for bit what `write` stores where nothing turns, else within a
derived bound of the formula in float64; and the store's operators together, as a decode loop uses them."""
import numpy as np
import pytest
import torch

from fathom_amd.rowstore8 import RowStore8
from oracle import rows8_oracle as R
from test_gpu_rows8 import BLK, DEV, _empty, _f32, _from_numpy, _garbage, _rand, _same
from test_gpu_rows8_multi import HALF, _check_chunk, _check_shared

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(BH, G, T, D, dtype, seed=0):
    q = _rand((BH * G, T, D), seed + 1, dtype).view(BH, G, T, D)
    return q, _rand((BH, T, D), seed + 2, dtype), _rand((BH, T, D), seed + 3, dtype)


def _inv(r, base=1e6):
    return torch.from_numpy(base ** (-np.arange(r // 2) * 2.0 / r)).float()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T, pos", [(1, 0), (1, 63), (5, 60), (64, 64), (200, 37), (333, 0)])
def test_without_weights_and_angles_it_is_write(code, dtype, D, T, pos):
    """Nothing turns: codes and scales are write's, the queries and keys come back as they are."""
    st, o = _garbage(2, 333, D, code)
    o["ks"][0], o["vs"][1] = 1e-4, 2e-3
    st = _from_numpy(o, code)
    q, K, V = _inputs(2, 3, T, D, dtype)
    out, keys = st.write_rotated(q.to(DEV), K.to(DEV), V.to(DEV), None, pos, keys=True)
    R.write(o, _f32(K), _f32(V), pos, code)
    _same(st, o, code)
    assert torch.equal(out.cpu(), q) and torch.equal(keys.cpu(), K)


def _turned_bound(x, t, inv, w, eps, half):
    """The formula's rows and the bound of their float32 evaluation, rounded to a type of half a step `half`.

    The sum of squares is a chain of 16 products and sums and up to 3 more; its root halves that, and the mean, root, inverse
    and two products add 6.  The angle left over is below 4 and rounded once (2^-23), its sine and cosine are off by two steps, and
    the turn has three roundings: with a pair's size h, 12 U h."""
    y = R.rotated(x, t, inv, w, eps)
    n = R.rotated(x, t, inv[:0], w, eps)
    h = np.abs(n)
    k = len(inv)
    pair = np.hypot(n[..., :k], n[..., k:2 * k])
    h[..., :k] = h[..., k:2 * k] = pair
    rel = (16 if w is not None else 0) * U
    tol = (rel + 12 * U) * h
    return y, tol + np.maximum(half * (np.abs(y) + tol), 2.0 ** -25 if half == 2.0 ** -11 else 0.0)  # steps of float16 end at 2^-24


def _stored_bound(y, tol, s, code):
    """Half a step of the format at y, and the bound of y itself: a code is the nearest to y / s of a scale s that is used
    as given; inverse and product round twice."""
    step = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) if code == "e4m3" else s * 0.5
    return (step + tol) * (1 + 4 * U) + 4 * U * np.abs(y)


@pytest.mark.parametrize("code, dtype, D", [("e4m3", torch.bfloat16, 128), ("int8", torch.float16, 64), ("int8", torch.float32, 128),
                                            ("e4m3", torch.float32, 64), ("e4m3", torch.float16, 128)])
@pytest.mark.parametrize("turn, norm", [(1.0, True), (1.0, False), (0.5, True), (0.25, False), (0.0, True)])
@pytest.mark.parametrize("G, T, offset", [(1, 1, 0), (7, 33, 100000), (4, 130, 2 ** 29), (3, 70, -20)])
def test_rotation(code, dtype, D, turn, norm, G, T, offset):
    BH, cap, eps = 3, 400, 1e-5
    q, K, V = _inputs(BH, G, T, D, dtype, seed=5)
    inv = _inv(int(D * turn)) if turn else None
    g = torch.Generator().manual_seed(9)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in "qk"]
    st, _ = _empty(BH, cap, D, code)
    pos = torch.tensor([0, 37, cap - T])
    on = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    out, keys = st.write_rotated(q.to(DEV), K.to(DEV), V.to(DEV), on(inv), pos.to(DEV), offset, on(w[0]), on(w[1]), eps, keys=True)
    alone, _ = _empty(BH, cap, D, code)
    alone.write(K.to(DEV), V.to(DEV), pos.to(DEV))
    assert torch.equal(st.v8.view(torch.uint8), alone.v8.view(torch.uint8)) and torch.equal(st.v_scale, alone.v_scale)
    ks = st.k_scale.double().cpu().numpy()
    values = R.values(st.k8.view(torch.uint8).cpu().numpy(), st.k_scale.cpu().numpy(), code)
    f = np.zeros(0) if inv is None else inv.double().numpy()
    ws = [None if x is None else x.double().numpy() for x in w]
    for b in range(BH):
        p = int(pos[b])
        t = p + offset + np.arange(T)
        y, tol = _turned_bound(q[b].double().numpy(), t, f, ws[0], eps, HALF[dtype])
        assert (np.abs(out[b].double().cpu().numpy() - y) <= tol).all()
        y, tol = _turned_bound(K[b].double().numpy(), t, f, ws[1], eps, HALF[dtype])
        assert (np.abs(keys[b].double().cpu().numpy() - y) <= tol).all()
        y, tol = _turned_bound(K[b].double().numpy(), t, f, ws[1], eps, 0.0)
        blocks = np.arange(p, p + T) // BLK
        s = ks[b][blocks][:, None]
        assert (np.abs(values[b, p:p + T] - y) <= _stored_bound(y, tol, s, code)).all()
        for blk in np.unique(blocks):
            a, e = np.abs(y[blocks == blk]).max() / R.qmax(code), tol[blocks == blk].max() / R.qmax(code)
            assert abs(ks[b][blk] - a) <= e + 2 * U * a
        assert not values[b, :p].any() and not values[b, p + T:].any()


def test_positions_are_those_of_the_prefix_and_the_row():
    """offset as an int, a tensor and inside pos give the same queries."""
    q, K, V = (x.to(DEV) for x in _inputs(2, 2, 5, 64, torch.float32))
    inv = _inv(64).to(DEV)
    a, b, c = (RowStore8.empty(2, 200, torch.int8, 64, DEV) for _ in range(3))
    first = a.write_rotated(q, K, V, inv, 100, 0)
    assert torch.equal(first, b.write_rotated(q, K, V, inv, 40, 60))
    assert torch.equal(first, c.write_rotated(q, K, V, inv, torch.tensor([40, 10], device=DEV), torch.tensor([60, 90], device=DEV)))
    assert torch.equal(b.read(40, 5, torch.float32)[0][0], c.read(torch.tensor([40, 10], device=DEV), 5, torch.float32)[0][0])


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_rows_that_do_not_fit_are_rotated_but_not_written(code):
    BH, cap, T, D = 5, 300, 90, 128
    st, o = _garbage(BH, cap, D, code)
    q, K, V = _inputs(BH, 2, T, D, torch.float32)
    inv = _inv(128)
    pos = torch.tensor([-1, 211, 300, 2 ** 31 - 1, -2 ** 31])
    out, keys = st.write_rotated(q.to(DEV), K.to(DEV), V.to(DEV), inv.to(DEV), pos.to(DEV), keys=True)
    _same(st, o, code, nan_payload=True)
    for b in range(BH):
        t = int(pos[b]) + np.arange(T)
        for got, x in ((out[b], q[b]), (keys[b], K[b])):
            y, tol = _turned_bound(x.double().numpy(), t, inv.double().numpy(), None, 0.0, HALF[torch.float32])
            if abs(int(pos[b])) > 2 ** 29:  # the angle itself is rounded in float64
                tol = tol + np.abs(x.double().numpy()).max() * 2.0 ** 32 * 2.0 ** -53
            assert (np.abs(got.double().cpu().numpy() - y) <= tol).all()


def test_values_that_are_not_finite():
    """NaN and infinities: a head's norm spreads them over its channels, the store takes them as write does."""
    q, K, V = _inputs(1, 2, 70, 128, torch.bfloat16)
    K[0, 3, 5], K[0, 66, 9], q[0, 1, 4, 7] = float("nan"), float("inf"), float("nan")
    V[0, 2, 2] = float("nan")
    w = torch.ones(128)
    st = RowStore8.empty(1, 70, torch.float8_e4m3fn, 128, DEV)
    out, keys = st.write_rotated(q.to(DEV), K.to(DEV), V.to(DEV), _inv(128).to(DEV), q_weight=w.to(DEV), k_weight=w.to(DEV), keys=True)
    bad = torch.zeros(70, dtype=torch.bool)
    bad[[3, 66]] = True
    assert torch.equal(keys[0].isnan().any(1).cpu(), bad) and torch.equal(out[0, 1].isnan().all(1).cpu(), torch.arange(70) == 4)
    k, v = st.read(0, 70)
    assert torch.equal(k[0].isnan().any(1).cpu(), bad) and int(v.isnan().sum()) == 1
    zeros = torch.zeros(1, 2, 70, 128, device=DEV)
    out = st.write_rotated(zeros, zeros[:, 0], zeros[:, 1], None, q_weight=w.to(DEV), k_weight=w.to(DEV))
    assert not out.any() and not st.k8.view(torch.uint8)[0].any()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("turn", [0.0, 0.25, 0.5])
def test_channels_that_do_not_turn_keep_their_own_values(code, dtype, D, turn):
    """Infinite and NaN channels behind r, or without a rotation, leave every other channel as it is, in the results and in the codes."""
    BH, G, T, r = 2, 3, 70, int(D * turn)
    q, K, V = _inputs(BH, G, T, D, dtype, seed=12)
    for x in (q[0, 1], q[1, 2], K[0], K[1]):
        x[3, r], x[4, r + 5], x[65, D - 1], x[66, D - 9], x[10, D // 2 + r // 2 + 1] = (float(v) for v in ("inf", "nan", "-inf", "nan", "inf"))
    st, o = _empty(BH, 100, D, code)
    out, keys = st.write_rotated(q.to(DEV), K.to(DEV), V.to(DEV), _inv(r).to(DEV) if r else None, 11, keys=True)
    for got, x in ((out, q), (keys, K)):
        torch.testing.assert_close(got[..., r:].cpu(), x[..., r:], rtol=0, atol=0, equal_nan=True)
        assert got[..., :r].isfinite().all()
    if dtype == torch.float32 or not r:  # the codes are made from these very keys
        R.write(o, _f32(keys.cpu()), _f32(V), 11, code)
        _same(st, o, code)


def test_layouts_and_weights_of_other_types():
    """Views of a fused projection, and whatever has to be copied first, give the bits of dense tensors."""
    BH, G, T, D = 1, 4, 50, 64
    q, K, V = (x.to(DEV) for x in _inputs(BH, G, T, D, torch.bfloat16))
    inv, w = _inv(64).to(DEV), torch.rand(64, device=DEV).bfloat16()
    st = [RowStore8.empty(BH, 64, torch.int8, D, DEV) for _ in range(5)]
    ref = st[0].write_rotated(q, K, V, inv, 3, q_weight=w, k_weight=w)
    qkv = torch.empty(T, G + 2, D, dtype=q.dtype, device=DEV)  # a token's heads side by side, as a fused projection has them
    qkv[:, :G], qkv[:, G], qkv[:, G + 1] = q[0].transpose(0, 1), K[0], V[0]
    views = qkv[:, :G].transpose(0, 1)[None], qkv[:, G][None], qkv[:, G + 1][None]
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    calls = [lambda s: s.write_rotated(*views, inv, 3, q_weight=w, k_weight=w), lambda s: s.write_rotated(odd, K, V, inv, 3, q_weight=w, k_weight=w),
             lambda s: s.write_rotated(q, K, V, inv.double(), torch.tensor([3], device=DEV), q_weight=w.float(), k_weight=w),
             lambda s: s.write_rotated(q, K, V, inv.repeat_interleave(2)[::2], 3, q_weight=w.double(), k_weight=w.double())]
    for f, s in zip(calls, st[1:]):
        assert torch.equal(f(s), ref)
        assert torch.equal(s.k8, st[0].k8) and torch.equal(s.v8, st[0].v8) and torch.equal(s.k_scale, st[0].k_scale)
    assert st[0].write_rotated(q[:, :, :0], K[:, :0], V[:, :0], inv).shape == (1, 4, 0, 64)


def test_refusals():
    st = RowStore8.empty(2, 100, torch.int8, 64, DEV)
    q, K, V = (x.to(DEV) for x in _inputs(2, 3, 10, 64, torch.bfloat16))
    inv, w = _inv(64).to(DEV), torch.ones(64, device=DEV)
    for bad in ((q[:1], K, V, inv), (q[:, :, :9], K, V, inv), (q[:, :0], K, V, inv), (q, K[:, :9], V, inv), (q, K, V.float(), inv),
                (q.float(), K, V, inv), (q[:, 0], K, V, inv), (q, K, V, inv[:20]), (q, K, V, torch.ones(64, device=DEV)), (q, K, V, inv[None]),
                (q, K, V, torch.ones(32, dtype=torch.int32, device=DEV)), (q.cpu(), K, V, inv), (q, K, V, inv.cpu())):
        with pytest.raises(ValueError):
            st.write_rotated(*bad)
    for kw in (dict(pos=91), dict(pos=-1), dict(offset=1 << 31), dict(offset=1 << 70), dict(q_weight=w[:32]), dict(k_weight=w.int()),
               dict(k_weight=w.cpu()), dict(eps=-1.0), dict(eps=float("nan")), dict(pos=torch.zeros(3, dtype=torch.int32, device=DEV)),
               dict(offset=torch.zeros(2, device=DEV))):
        with pytest.raises(ValueError):
            st.write_rotated(q, K, V, inv, **kw)
    assert not st.k8.any() and not st.v_scale.any()


# ----------------------------------------------------------------------------- together
def _copy(st):
    return {"k8": st.k8.view(torch.uint8).cpu().numpy(), "v8": st.v8.view(torch.uint8).cpu().numpy(), "ks": st.k_scale.cpu().numpy(),
            "vs": st.v_scale.cpu().numpy()}


def test_a_batch_from_prompt_to_tokens():
    """Sequences behind a shared prompt: the prompt's chunks are rotated, stored and attended to; then each sequence's tokens,
    over prompt and own tokens, with a layer of windows beside it; in a graph whose places change between replays."""
    B, H, G, D, P, chunk = 3, 2, 4, 128, 300, 128
    inv, w = _inv(D).to(DEV), (1 + 0.1 * torch.randn(2, D, generator=torch.Generator().manual_seed(1))).to(DEV)
    prompt = RowStore8.empty(H, P, torch.float8_e4m3fn, D, DEV)
    whole = RowStore8.empty(B * H, P + 40, torch.float8_e4m3fn, D, DEV)  # the same, a row for each sequence
    q, K, V = (x.to(DEV) for x in _inputs(H, G, P, D, torch.bfloat16, seed=30))
    for p in range(0, P, chunk):
        part = slice(p, min(P, p + chunk))
        args = (q[:, :, part], K[:, part], V[:, part])
        rot = prompt.write_rotated(*args, inv, p, q_weight=w[0], k_weight=w[1])
        many = [x.repeat(B, *[1] * (x.dim() - 1)) for x in args]
        again = whole.write_rotated(*many, inv, p, q_weight=w[0], k_weight=w[1])
        assert torch.equal(again[:H], rot)
        end = min(P, p + chunk)
        o = _copy(prompt)
        _check_chunk(prompt.chunk_attention(rot, end), rot.cpu(), o, "e4m3", [end] * H, every=31)
    own = RowStore8.empty(B * H, 40, torch.float8_e4m3fn, D, DEV)
    pos = torch.zeros(B * H, dtype=torch.int32, device=DEV)
    step = [x.to(DEV) for x in _inputs(B * H, G, 1, D, torch.bfloat16, seed=40)]

    def decode():
        rot = own.write_rotated(*step, inv, pos, P, q_weight=w[0], k_weight=w[1])[:, :, 0]
        return rot, own.shared_attention(rot, pos + 1, prompt, P), own.attention(rot, pos + 1, window=8, sinks=2)

    decode()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = decode()
    for i in range(20):
        for x, new in zip(step, _inputs(B * H, G, 1, D, torch.bfloat16, seed=50 + 4 * i)):
            x.copy_(new)
        pos.fill_(i)
        graph.replay()
        rot = whole.write_rotated(*step, inv, P + i, q_weight=w[0], k_weight=w[1])[:, :, 0]
        assert torch.equal(rot, outs[0])
        if i % 6 == 0:
            o = _copy(own)
            _check_shared(outs[1], rot.cpu(), o, _copy(prompt), "e4m3", [i + 1] * B * H, [P] * H)
            k, v = R.values(o["k8"], o["ks"], "e4m3"), R.values(o["v8"], o["vs"], "e4m3")
            for r in range(B * H):
                for g in range(G):
                    ref, tol = R.attention(rot[r, g].double().cpu().numpy(), k[r], v[r], R.sees(i, i + 1, 8, 2), i + 1, D ** -0.5)
                    assert (np.abs(outs[2][r, g].double().cpu().numpy() - ref) <= tol).all()


def test_offsets_beyond_32_bits():
    """An int is refused, a tensor's values count as the nearest of 32 bits."""
    q, K, V = (x.to(DEV) for x in _inputs(2, 2, 5, 64, torch.float32))
    inv = _inv(64).to(DEV)
    st = RowStore8.empty(2, 200, torch.int8, 64, DEV)
    with pytest.raises(ValueError):
        st.write_rotated(q, K, V, inv, 0, 1 << 31)
    far, near = torch.tensor([1 << 40, -(1 << 40)], device=DEV), torch.tensor([(1 << 31) - 1, -(1 << 31)], device=DEV)
    assert torch.equal(st.write_rotated(q, K, V, inv, 0, far), st.write_rotated(q, K, V, inv, 0, near))
