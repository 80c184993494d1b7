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


class RowStore8:
    """The K/V rows of one layer in 8 bits; see the module's text.

    k8, v8 [BH, cap, d] (d = 64 or 128; float8_e4m3fn or int8), k_scale, v_scale
    [BH, ceil(cap / 64)] float32: contiguous, on one GPU.  They are the store: it
    keeps nothing else, and methods write into them."""

    def __init__(self, k8, v8, k_scale, v_scale):
        shape, dev = k8.shape, k8.device
        if dev.type != "cuda":
            _need_gpu(k8)
        if len(shape) != 3 or k8.dtype not in _CODES or shape[2] not in (64, 128):
            raise ValueError(f"codes must be float8_e4m3fn or int8 [BH, cap, 64 or 128], got {k8.dtype} {tuple(shape)}")
        self.BH, self.cap, self.d = shape
        if v8.shape != shape or v8.dtype != k8.dtype:
            raise ValueError(f"v8 {v8.dtype} {tuple(v8.shape)} must be like k8 {k8.dtype} {tuple(shape)}")
        scales = (self.BH, -(-self.cap // BLK))
        if k_scale.shape != scales or v_scale.shape != scales or k_scale.dtype != _F32 or v_scale.dtype != _F32:
            raise ValueError(f"scales must be float32 {list(scales)}, got {k_scale.dtype} {tuple(k_scale.shape)} and "
                             f"{v_scale.dtype} {tuple(v_scale.shape)}")
        if not (v8.device == k_scale.device == v_scale.device == dev and k8.is_contiguous() and v8.is_contiguous()
                and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("the store's tensors must be contiguous and on one device")
        self.k8, self.v8, self.k_scale, self.v_scale = k8, v8, k_scale, v_scale
        self.device = dev
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
        dev = self.device.index
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
        if v.device != self.device:
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
        if q.device != self.device:
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
        return q, at, self.d ** -0.5 if scale is None else float(scale), softcap, slopes

    def _workspace(self, query, G, positions):
        """The call's workspace (or None), its address and size, for at least `positions`: sizes grow with them, so one query
        serves up to the next power of two."""
        if positions < 1:
            return None, None, 0
        bits = (positions - 1).bit_length()
        key = query, self.BH, G, self.d, bits
        nbytes = _SIZES.get(key)
        if nbytes is None:
            nbytes = _SIZES[key] = getattr(_lib.lib(), query)(self.BH, G, self.d, 1 << bits)
        if not nbytes:
            return None, None, 0
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=self.device)
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

    def _read(self, idx_at, rows_at, at, R, dtype):
        if dtype not in _KDT:
            raise ValueError(f"dtype {dtype} unsupported (float32, float16, bfloat16)")
        if R < 0:
            raise ValueError(f"{R} tokens")
        K = torch.empty((self.BH, R, self.d), dtype=dtype, device=self.device)
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
    def attention(self, q, length, window=0, scale=None, softcap=None, slopes=None):
        """Attention of one token per row, q [BH, G, d] (float32, float16 or bfloat16),
        over the row's first `length` tokens, or the last `window` of them (0: all):
        softmax(z) . V in float32 [BH, G, d], with
          z_t = scale q . K_t, capped to softcap tanh(z_t / softcap) if softcap is given,
                then biased by slopes[bh, g] (t - (length - 1)) if slopes are given
        (slopes [BH, G], or [G]; scale defaults to d ** -0.5; a cap below 2^-64 counts as
        that, one above 2^90 as none).  A tensor length is taken
        as within [0, cap].  A row without tokens gives zeros."""
        q, q_at, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        lens, lens_at, n = self._per_row(length, "length")
        G, window = q.shape[1], max(min(int(window), _FAR), -1)  # the library refuses negative ones
        positions = n if lens is None else self.cap
        positions = max(min(positions, window) if window > 0 else positions, 0)
        ws, ws_at, nbytes = self._workspace("fathom_rows8_attention_workspace_bytes", G, positions)
        out = torch.empty_like(q, dtype=_F32)
        self._call("fathom_rows8_attention", q_at, _KDT[q.dtype], *self._store(), self._code, self.BH, G, self.d, self.cap,
                   lens_at, n, window, scale, softcap, None if slopes is None else slopes.data_ptr(), out.data_ptr(), ws_at,
                   nbytes)
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
