"""K/V rows in 8 bits, and attention over them.

The key index (bitplane.PlaneStore) ends in K/V rows.  In bf16 a token of one
(batch, KV head) row takes 512 bytes (D = 128); here it takes 256, and 1/8 for its
block's scales, so the rows of long sequences stay in HBM beside the index, and
attention over them reads half the bytes.  It has no counterpart in the
reference.

RowStore8 keeps, per row and for K and V apart, codes [BH, cap, d]
(torch.float8_e4m3fn or torch.int8) and one float32 scale per 64-token block
[BH, ceil(cap / 64)]: value = code * scale.  The caller keeps the lengths: `pos` and
`length` are ints, or int32 tensors [BH] on the device for rows of different
lengths (also in captured graphs, where they change between replays).  Calls run
asynchronously on the device's current stream.
"""
import math

import torch

from . import _lib
from .bitplane import BLK, D, _KDT, _need_gpu

__all__ = ["RowStore8"]

_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64
_SHORT = {_I32, torch.int16, torch.uint16, torch.int8, torch.uint8}
_FAR = 1 << 62  # ctypes would wrap what is longer
_SIZES = {}  # workspace bytes by query and shape
_CODES = {torch.float8_e4m3fn: _lib.DT_E4M3, torch.int8: _lib.DT_I8}


def _rows(x):
    """Rows [BH, T, d] of a float type as the kernels read them, with their strides: any,
    but dense rows, each at a multiple of 16 bytes (a copy is made of others)."""
    if x.dtype in _KDT and x.is_contiguous() and not x.data_ptr() & 15:
        _, T, d = x.shape
        return x, T * d, d
    if x.dtype not in _KDT:
        x = x.float()
    size = 4 if x.dtype == _F32 else 2
    BH, T, _ = x.shape
    sr, st, sd = x.stride()
    sr, st = sr if BH > 1 else 0, st if T > 1 else 0  # the stride of a single row says nothing
    if sd != 1 or (x.data_ptr() | sr * size | st * size) & 15:
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        sr, st, _ = x.stride()
    return x, sr, st


def _heads(q):
    """Queries [BH, G, T, d] of a float type, with the strides of rows, heads and tokens: any, but dense channels, each
    at a multiple of 16 bytes (a copy is made of others)."""
    if q.dtype in _KDT and q.is_contiguous() and not q.data_ptr() & 15:
        _, G, T, d = q.shape
        return q, G * T * d, T * d, d
    if q.dtype not in _KDT:
        q = q.float()
    size = 4 if q.dtype == _F32 else 2
    (BH, G, T, _), (sr, sh, st, sd) = q.shape, q.stride()
    sr, sh, st = sr if BH > 1 else 0, sh if G > 1 else 0, st if T > 1 else 0  # the stride of a single one says nothing
    if sd != 1 or (q.data_ptr() | sr * size | sh * size | st * size) & 15:
        q = torch.empty(q.shape, dtype=q.dtype, device=q.device).copy_(q)
        sr, sh, st, _ = q.stride()
    return q, sr, sh, st


class RowStore8:
    """The K/V rows of one layer in 8 bits; see the module's text.

    k8, v8 [BH, cap, d] (d = 64 or 128; float8_e4m3fn or int8), k_scale, v_scale
    [BH, ceil(cap / 64)] float32: contiguous, on one GPU.  They are the store: it
    keeps nothing else, and methods write into them."""

    def __init__(self, k8, v8, k_scale, v_scale):
        shape, dev, gpu = k8.shape, k8.device, k8.get_device()
        if gpu < 0:
            _need_gpu(k8)
        if len(shape) != 3 or k8.dtype not in _CODES or shape[2] not in (64, 128):
            raise ValueError(f"codes must be float8_e4m3fn or int8 [BH, cap, 64 or 128], got {k8.dtype} {tuple(shape)}")
        self.BH, self.cap, self.d = shape
        if v8.shape != shape or v8.dtype != k8.dtype:
            raise ValueError(f"v8 {v8.dtype} {tuple(v8.shape)} must be like k8 {k8.dtype} {tuple(shape)}")
        scales = (shape[0], -(-shape[1] // BLK))
        if k_scale.shape != scales or v_scale.shape != scales or k_scale.dtype != _F32 or v_scale.dtype != _F32:
            raise ValueError(f"scales must be float32 {list(scales)}, got {k_scale.dtype} {tuple(k_scale.shape)} and "
                             f"{v_scale.dtype} {tuple(v_scale.shape)}")
        if not (v8.get_device() == k_scale.get_device() == v_scale.get_device() == gpu and k8.is_contiguous() and v8.is_contiguous()
                and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("the store's tensors must be contiguous and on one device")
        self.k8, self.v8, self.k_scale, self.v_scale = k8, v8, k_scale, v_scale
        self.device, self._gpu = dev, gpu
        self._code = _CODES[k8.dtype]

    @classmethod
    def empty(cls, BH, cap, dtype=torch.float8_e4m3fn, d=D, device=None):
        """A store of BH rows with room for cap tokens, all zeros."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        k8, v8 = (torch.zeros(BH, cap, d, dtype=torch.uint8, device=dev).view(dtype) for _ in "kv")
        ks, vs = (torch.zeros(BH, -(-cap // BLK), dtype=torch.float32, device=dev) for _ in "kv")
        return cls(k8, v8, ks, vs)

    # ------------------------------------------------------------------ arguments
    # A call of a few tokens is as long as its host side, so arguments go to the
    # library as plain ints and are checked without building objects.
    def _call(self, name, *args):
        """The entry point on the store's device and its current stream."""
        dev = self._gpu
        fn = getattr(_lib.lib(), name)
        if _current_device() == dev:
            rc = fn(*args, _raw_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = fn(*args, _raw_stream(dev))
        if rc:
            _lib.check(rc, name)

    def _store(self):
        return self.k8.data_ptr(), self.v8.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()

    def _elsewhere(self, t):
        _need_gpu(t)
        raise ValueError(f"a tensor on {t.device}, the store is on {self.device}")

    def _per_row(self, v, what):
        """A per-row argument as (int32 tensor or None, its address, int)."""
        if not isinstance(v, torch.Tensor):
            v = int(v)
            if not -_FAR < v < _FAR:
                raise ValueError(f"{what} {v}")
            return None, None, v
        if v.get_device() != self._gpu:
            self._elsewhere(v)
        dtype = v.dtype
        if v.shape != (self.BH,) or (dtype != _I32 and (dtype.is_floating_point or dtype.is_complex or dtype == torch.bool)):
            raise ValueError(f"{what} must be an int or integers [{self.BH}], got {dtype} {tuple(v.shape)}")
        if dtype != _I32 or not v.is_contiguous():
            if dtype not in _SHORT:  # places beyond int32 stay beyond every store
                if dtype == torch.uint64:
                    v = v.view(_I64)
                    v = v.masked_fill(v < 0, _FAR)
                v = v.to(_I64).clamp(-(1 << 31), (1 << 31) - 1)
            v = v.to(_I32).contiguous()
        return v, v.data_ptr(), 0

    def _query(self, q, scale, softcap, slopes):
        """q as the kernels read it, with its address; the scale, cap and slopes of a call."""
        if q.get_device() != self._gpu:
            self._elsewhere(q)
        shape = q.shape
        if len(shape) != 3 or shape[0] != self.BH or shape[2] != self.d or shape[1] < 1:
            raise ValueError(f"q {tuple(shape)} must be [{self.BH}, G, {self.d}]")
        if q.dtype not in _KDT or not q.is_contiguous():
            q = (q if q.dtype in _KDT else q.float()).contiguous()
        at = q.data_ptr()
        if at % 16:
            q = q.clone()
            at = q.data_ptr()
        return q, at, *self._scores(shape, scale, softcap, slopes)

    def _scores(self, shape, scale, softcap, slopes):
        """The scale, cap and slopes of a call whose queries have this shape."""
        softcap = 0.0 if softcap is None else float(softcap)
        if not 0.0 <= softcap < math.inf:
            raise ValueError(f"softcap {softcap} must be positive and finite (None or 0: no cap)")
        if softcap:  # float32 would make 0 or infinity of others
            softcap = min(max(softcap, 1e-30), 1e30)
        if slopes is not None:
            if slopes.device != self.device:
                self._elsewhere(slopes)
            if slopes.dtype != _F32 or slopes.shape != shape[:2] or not slopes.is_contiguous():
                slopes = slopes.float().expand(shape[:2]).contiguous()
        return self.d ** -0.5 if scale is None else float(scale), softcap, slopes

    def _workspace(self, query, G, positions, *queries):
        """The call's workspace (or None), its address and size, for at least `positions`: sizes grow with them, so one query
        serves up to the next power of two."""
        if positions < 1:
            return None, None, 0
        bits = (positions - 1).bit_length()
        key = query, self.BH, G, *queries, self.d, bits
        nbytes = _SIZES.get(key)
        if nbytes is None:
            nbytes = _SIZES[key] = getattr(_lib.lib(), query)(self.BH, G, *queries, self.d, 1 << bits)
        if not nbytes:
            return None, None, 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return ws, ws.data_ptr(), nbytes

    # ------------------------------------------------------------------ writing and reading
    def write(self, K, V, pos=0):
        """Quantise K, V [BH, T, d] into tokens pos .. pos + T - 1 of each row: a
        prompt, a piece of one, or one step's token.

        A 64-token block's scale is its largest finite |x| / 448 (e4m3) or 127 (int8); a
        block that holds earlier tokens keeps its scale and its sign, or takes the least
        power-of-two multiple of it that holds the new tokens, to which its earlier
        codes are then rounded.  Tokens at pos + T and behind are no longer the row's.
        With a tensor `pos`, rows whose tokens do not all fit into the store (a negative
        pos among them) are left as they are; an int pos that does not fit raises.  K
        and V may be views with any strides (their rows dense)."""
        for t in (K, V):
            if t.device != self.device:
                self._elsewhere(t)
        if K.dim() != 3 or K.shape != V.shape or K.shape[0] != self.BH or K.shape[2] != self.d or K.dtype != V.dtype:
            raise ValueError(f"K {K.dtype} {tuple(K.shape)} and V {V.dtype} {tuple(V.shape)} must be alike, "
                             f"[{self.BH}, T, {self.d}]")
        rows, rows_at, at = self._per_row(pos, "pos")
        K, kr, kt = _rows(K)
        V, vr, vt = _rows(V)
        self._call("fathom_rows8_write", K.data_ptr(), V.data_ptr(), _KDT[K.dtype], kr, kt, vr, vt, rows_at, at, self.BH,
                   K.shape[1], self.d, self.cap, self._code, *self._store())

    def write_rotated(self, q, K, V, inv_freq, pos=0, offset=0, q_weight=None, k_weight=None, eps=1e-6, keys=False):
        """What a layer does with its projections, in one pass: norms of each query and key head, the position rotation,
        and `write` of the rotated keys and of V.  q [BH, G, T, d], K, V [BH, T, d], all of one type.  Returns the
        rotated queries [BH, G, T, d], or with keys=True (queries, keys [BH, T, d]), both of q's type; the store's codes are
        made from the keys before that rounding.

        With weights (q_weight, k_weight [d]; None: no norm) x becomes x / sqrt(mean(x^2) + eps) * weight.  Token i
        of a row stands at position t = pos + i + offset; with inv_freq [r / 2] (float32, finite and below 2^50 in size;
        r <= d a multiple of 16; None: no rotation) channels c and c + r / 2 become (x_c cos - x_{c+r/2} sin,
        x_{c+r/2} cos + x_c sin) of the angle t inv_freq[c], whose whole turns are dropped exactly at any t; channels
        behind r stay.  offset is an int or integers [BH]: what stands before the store's first token, as a shared prefix
        does, of 32 bits (of a tensor's others the nearest).  Types other than float32, float16 and bfloat16 are taken, and given
        back, as float32.  Views as in `write`; with a tensor `pos`, rows whose tokens do not all fit are rotated but not written."""
        gpu, BH, d = self._gpu, self.BH, self.d
        for t in (q, K, V):
            if t.get_device() != gpu:
                self._elsewhere(t)
        shape, k_shape, dtype = q.shape, K.shape, q.dtype
        if len(k_shape) != 3 or k_shape != V.shape or k_shape[0] != BH or k_shape[2] != d:
            raise ValueError(f"K {tuple(k_shape)} and V {tuple(V.shape)} must be alike, [{BH}, T, {d}]")
        T = k_shape[1]
        if len(shape) != 4 or shape[0] != BH or shape[1] < 1 or shape[2] != T or shape[3] != d:
            raise ValueError(f"q {tuple(shape)} must be [{BH}, G, {T}, {d}]")
        if not dtype == K.dtype == V.dtype or not dtype.is_floating_point:
            raise ValueError(f"q {dtype}, K {K.dtype} and V {V.dtype} must be of one float type")
        turned, inv_at = 0, None
        if inv_freq is not None:
            if inv_freq.get_device() != gpu:
                self._elsewhere(inv_freq)
            turned = 2 * inv_freq.numel()
            if inv_freq.dim() != 1 or turned > d or turned % 16 or not inv_freq.dtype.is_floating_point:
                raise ValueError(f"inv_freq {inv_freq.dtype} {tuple(inv_freq.shape)} must be float32 [r / 2], r <= {d} a multiple of 16")
            if inv_freq.dtype != _F32 or not inv_freq.is_contiguous():
                inv_freq = inv_freq.float().contiguous()
            inv_at = inv_freq.data_ptr()
        w_dtype, q_weight_at, k_weight_at = _F32, None, None
        if q_weight is not None or k_weight is not None:
            first, last = k_weight if q_weight is None else q_weight, q_weight if k_weight is None else k_weight
            if first.dtype == last.dtype and first.dtype in _KDT:
                w_dtype = first.dtype
            if q_weight is not None:
                q_weight = self._weight(q_weight, w_dtype)
                q_weight_at = q_weight.data_ptr()
            if k_weight is not None:
                k_weight = self._weight(k_weight, w_dtype)
                k_weight_at = k_weight.data_ptr()
        eps = float(eps)
        if not 0.0 <= eps < math.inf:
            raise ValueError(f"eps {eps} must be finite and not negative")
        rows, rows_at, at = self._per_row(pos, "pos")
        shifts, shifts_at, shift = self._per_row(offset, "offset")
        q, qr, qh, qt = _heads(q)
        K, kr, kt = _rows(K)
        V, vr, vt = _rows(V)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = torch.empty_like(K, memory_format=torch.contiguous_format) if keys else None
        self._call("fathom_rows8_write_rotated", q.data_ptr(), K.data_ptr(), V.data_ptr(), _KDT[q.dtype], qr, qh, qt, kr, kt, vr,
                   vt, rows_at, at, shifts_at, shift, inv_at, turned, q_weight_at, k_weight_at, _KDT[w_dtype], eps, BH, shape[1], T,
                   d, self.cap, self._code, *self._store(), out.data_ptr(), None if k_out is None else k_out.data_ptr())
        return (out, k_out) if keys else out

    def _weight(self, w, dtype):
        """A norm's weights as the kernel reads them."""
        if w.get_device() != self._gpu:
            self._elsewhere(w)
        if w.shape != (self.d,) or not w.dtype.is_floating_point:
            raise ValueError(f"a weight {w.dtype} {tuple(w.shape)} must be floats [{self.d}]")
        return w if w.dtype == dtype and w.is_contiguous() else w.to(dtype).contiguous()

    def _read(self, idx_at, rows_at, at, R, dtype):
        if dtype not in _KDT:
            raise ValueError(f"dtype {dtype} unsupported (float32, float16, bfloat16)")
        if R < 0:
            raise ValueError(f"{R} tokens")
        K = torch.empty(self.BH, R, self.d, dtype=dtype, device=self.device)
        V = torch.empty_like(K)
        self._call("fathom_rows8_read", *self._store(), self._code, self.BH, self.cap, self.d, idx_at, rows_at, at, R,
                   _KDT[dtype], K.data_ptr(), V.data_ptr())
        return K, V

    def read(self, pos, T, dtype=torch.bfloat16):
        """The values of tokens pos .. pos + T - 1 of each row, K, V [BH, T, d];
        tokens outside the store are zeros."""
        rows, rows_at, at = self._per_row(pos, "pos")
        return self._read(None, rows_at, at, int(T), dtype)

    def gather_rows(self, idx, dtype=torch.bfloat16):
        """The values of the listed tokens idx [BH, R], K, V [BH, R, d]; tokens outside
        the store give zero rows, as offload.gather_rows does."""
        if idx.device != self.device:
            self._elsewhere(idx)
        if idx.dim() != 2 or idx.shape[0] != self.BH:
            raise ValueError(f"idx {tuple(idx.shape)} must be [{self.BH}, R]")
        if idx.dtype != _I64 or not idx.is_contiguous():
            idx = idx.to(_I64).contiguous()
        return self._read(idx.data_ptr(), None, 0, idx.shape[1], dtype)

    # ------------------------------------------------------------------ attention
    def attention(self, q, length, window=0, scale=None, softcap=None, slopes=None, sinks=0):
        """Attention of one token per row, q [BH, G, d] (float32, float16 or bfloat16),
        over the row's first `length` tokens, or the last `window` of them (0: all) and the first `sinks`:
        softmax(z) . V in float32 [BH, G, d], with
          z_t = scale q . K_t, capped to softcap tanh(z_t / softcap) if softcap is given,
                then biased by slopes[bh, g] (t - (length - 1)) if slopes are given
        (slopes [BH, G], or [G]; scale defaults to d ** -0.5; a cap below 2^-64 counts as
        that, one above 2^90 as none).  A tensor length is taken
        as within [0, cap].  A row without tokens gives zeros."""
        q, q_at, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        lens, lens_at, n = self._per_row(length, "length")
        G, window, sinks = q.shape[1], max(min(int(window), _FAR), -1), max(min(int(sinks), _FAR), -1)  # the library refuses negative ones
        positions = n if lens is None else self.cap
        positions = max(min(positions, window + -(-sinks // BLK) * BLK) if window > 0 else positions, 0)
        ws, ws_at, nbytes = self._workspace("fathom_rows8_attention_workspace_bytes", G, positions)
        out = torch.empty_like(q, dtype=_F32)
        extra = (sinks,) if sinks else ()
        self._call("fathom_rows8_sink_attention" if sinks else "fathom_rows8_attention", q_at, _KDT[q.dtype], *self._store(),
                   self._code, self.BH, G, self.d, self.cap, lens_at, n, window, *extra, scale, softcap,
                   None if slopes is None else slopes.data_ptr(), out.data_ptr(), ws_at, nbytes)
        return out

    def gather_attention(self, q, idx, length=None, scale=None, softcap=None, slopes=None):
        """The same attention over the selected tokens idx [BH, G, k] (as
        PlaneStore.scan_topk gives them): [BH, G, d] float32.  A token listed twice counts
        twice.  Tokens outside [0, length) (length defaults to cap) take no part, so a
        selection may be padded with -1 (offload.gather_attention's zero rows score 0
        instead)."""
        q, q_at, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        if idx.device != self.device:
            self._elsewhere(idx)
        G = q.shape[1]
        shape = idx.shape
        if len(shape) != 3 or shape[0] != self.BH or shape[1] != G:
            raise ValueError(f"idx {tuple(idx.shape)} must be [{self.BH}, {G}, k]")
        if idx.dtype != _I64 or not idx.is_contiguous():
            idx = idx.to(_I64).contiguous()
        k = shape[2]
        lens, lens_at, n = self._per_row(self.cap if length is None else length, "length")
        ws, ws_at, nbytes = self._workspace("fathom_rows8_gather_attention_workspace_bytes", G, k)
        out = torch.empty_like(q, dtype=_F32)
        self._call("fathom_rows8_gather_attention", q_at, _KDT[q.dtype], idx.data_ptr(), *self._store(), self._code, self.BH, G,
                   k, self.d, self.cap, lens_at, n, scale, softcap, None if slopes is None else slopes.data_ptr(),
                   out.data_ptr(), ws_at, nbytes)
        return out

    def chunk_attention(self, q, length, window=0, sinks=0, scale=None, softcap=None, slopes=None):
        """Attention of the last T tokens of each row, q [BH, G, T, d] (float32, float16 or bfloat16, any strides), each
        over the tokens up to its own: a prompt, a piece of one, or drafted tokens, once `write` or `write_rotated` has
        their keys and values.  Token i of a row of `length` tokens stands at place p = length - T + i and sees tokens
        t <= p, with a window only the last `window` of them and the first `sinks`.  Scores as in `attention`, with the
        bias slopes[bh, g] (t - p); the scale is at most 2^127 in size, here and in `shared_attention`.  [BH, G, T, d] in
        q's type (float32 for types other than those three); a token before the row's first (p < 0) gives zeros, so rows of
        fewer than T tokens are padded in front."""
        if q.get_device() != self._gpu:
            self._elsewhere(q)
        shape = q.shape
        if len(shape) != 4 or shape[0] != self.BH or shape[1] < 1 or shape[3] != self.d:
            raise ValueError(f"q {tuple(shape)} must be [{self.BH}, G, T, {self.d}]")
        scale, softcap, slopes = self._scores(shape, scale, softcap, slopes)
        lens, lens_at, n = self._per_row(length, "length")
        q, qr, qh, qt = _heads(q)
        G, T = shape[1], shape[2]
        window, sinks = max(min(int(window), _FAR), -1), max(min(int(sinks), _FAR), -1)
        positions = n if lens is None else self.cap
        positions = max(min(positions, window + T + -(-sinks // BLK) * BLK) if window > 0 else positions, 0)
        ws, ws_at, nbytes = self._workspace("fathom_rows8_chunk_attention_workspace_bytes", G, positions, T)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        self._call("fathom_rows8_chunk_attention", q.data_ptr(), _KDT[q.dtype], qr, qh, qt, *self._store(), self._code, self.BH, G, T,
                   self.d, self.cap, lens_at, n, window, sinks, scale, softcap, None if slopes is None else slopes.data_ptr(),
                   out.data_ptr(), ws_at, nbytes)
        return out

    def shared_attention(self, q, length, prefix, prefix_length, scale=None, softcap=None, slopes=None):
        """`attention` for a batch whose sequences begin with the same tokens: `prefix`, a RowStore8 of H rows, holds
        them once, this store's rows [B, H] hold what follows (`length` tokens, ints or integers [B H]).  Row (b, h) attends to
        the first prefix_length (int, or integers [H]) tokens of the prefix's row h and then its own, in one
        softmax; the prefix is read once for all B.  One token a row: several behind a prefix need it in their own rows.
        q [B H, G, d]; [B H, G, d] float32."""
        if not isinstance(prefix, RowStore8) or prefix.device != self.device:
            raise ValueError(f"the prefix must be a RowStore8 on {self.device}")
        H = prefix.BH
        if not H or prefix.d != self.d or prefix._code != self._code or self.BH % H:
            raise ValueError(f"a prefix of {H} rows of {prefix.d} {prefix.k8.dtype} codes does not fit {self.BH} rows of "
                             f"{self.d} {self.k8.dtype}")
        q, q_at, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        lens, lens_at, n = self._per_row(length, "length")
        plens, plens_at, pn = prefix._per_row(prefix_length, "prefix_length")
        G = q.shape[1]
        bits = [max(min(v, _FAR), 1) - 1 for v in (pn if plens is None else prefix.cap, n if lens is None else self.cap)]
        key = "shared", H, self.BH, G, self.d, bits[0].bit_length(), bits[1].bit_length()
        nbytes = _SIZES.get(key)
        if nbytes is None:
            nbytes = _SIZES[key] = _lib.lib().fathom_rows8_shared_attention_workspace_bytes(
                H, self.BH // H, G, self.d, 1 << bits[0].bit_length(), 1 << bits[1].bit_length())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        out = torch.empty_like(q, dtype=_F32)
        self._call("fathom_rows8_shared_attention", q_at, _KDT[q.dtype], *prefix._store(), H, prefix.cap, plens_at, pn,
                   *self._store(), self._code, self.BH // H, G, self.d, self.cap, lens_at, n, scale, softcap,
                   None if slopes is None else slopes.data_ptr(), out.data_ptr(), ws.data_ptr(), nbytes)
        return out
