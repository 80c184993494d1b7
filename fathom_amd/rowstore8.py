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
import torch

from . import _lib
from .bitplane import BLK, D, _KDT, _need_gpu, _ptr, _stream

__all__ = ["RowStore8"]

_CODES = {torch.float8_e4m3fn: _lib.DT_E4M3, torch.int8: _lib.DT_I8}


def _aligned(x):
    """Rows [BH, T, d] of a float type as the kernels read them: any strides, but dense
    rows, and every row at a multiple of 16 bytes (a copy is made of others)."""
    if x.dtype not in _KDT:
        x = x.float()
    size = x.element_size()
    if x.stride(2) != 1 or x.data_ptr() % 16 or x.stride(0) * size % 16 or x.stride(1) * size % 16:
        x = x.contiguous()
        x = x.clone() if x.data_ptr() % 16 else x
    return x


class RowStore8:
    """The K/V rows of one layer in 8 bits; see the module's text.

    k8, v8 [BH, cap, d] (d = 64 or 128; float8_e4m3fn or int8), k_scale, v_scale
    [BH, ceil(cap / 64)] float32: contiguous, on one GPU.  They are the store: it
    keeps nothing else, and methods write into them."""

    def __init__(self, k8, v8, k_scale, v_scale):
        _need_gpu(k8, v8, k_scale, v_scale)
        if k8.dim() != 3 or k8.dtype not in _CODES or k8.shape[2] not in (64, 128):
            raise ValueError(f"codes must be float8_e4m3fn or int8 [BH, cap, 64 or 128], got {k8.dtype} {tuple(k8.shape)}")
        self.BH, self.cap, self.d = k8.shape
        if v8.shape != k8.shape or v8.dtype != k8.dtype:
            raise ValueError(f"v8 {v8.dtype} {tuple(v8.shape)} must be like k8 {k8.dtype} {tuple(k8.shape)}")
        nblk = -(-self.cap // BLK)
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != (self.BH, nblk):
                raise ValueError(f"scales must be float32 [{self.BH}, {nblk}], got {s.dtype} {tuple(s.shape)}")
        for t in (k8, v8, k_scale, v_scale):
            if not t.is_contiguous() or t.device != k8.device:
                raise ValueError("the store's tensors must be contiguous and on one device")
        self.k8, self.v8, self.k_scale, self.v_scale = k8, v8, k_scale, v_scale
        self.device = k8.device
        self._code = _CODES[k8.dtype]

    @classmethod
    def empty(cls, BH, cap, dtype=torch.float8_e4m3fn, d=D, device=None):
        """A store of BH rows with room for cap tokens, all zeros."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        k8, v8 = (torch.zeros(BH, cap, d, dtype=torch.uint8, device=dev).view(dtype) for _ in "kv")
        ks, vs = (torch.zeros(BH, -(-cap // BLK), dtype=torch.float32, device=dev) for _ in "kv")
        return cls(k8, v8, ks, vs)

    # ------------------------------------------------------------------ arguments
    def _call(self, name, *args):
        """The entry point on the store's device and its current stream."""
        if torch.cuda.current_device() == self.device.index:
            _lib.call(name, *args, _stream(self.device))
        else:
            with torch.cuda.device(self.device):
                _lib.call(name, *args, _stream(self.device))

    def _tensors(self):
        return _ptr(self.k8), _ptr(self.v8), _ptr(self.k_scale), _ptr(self.v_scale)

    def _here(self, *tensors):
        _need_gpu(*tensors)
        for t in tensors:
            if t.device != self.device:
                raise ValueError(f"a tensor on {t.device}, the store is on {self.device}")

    def _per_row(self, v, what):
        """A per-row argument as (int32 tensor or None, int)."""
        if not torch.is_tensor(v):
            return None, int(v)
        self._here(v)
        if v.shape != (self.BH,) or v.dtype.is_floating_point or v.dtype == torch.bool:
            raise ValueError(f"{what} must be an int or integers [{self.BH}], got {v.dtype} {tuple(v.shape)}")
        if v.dtype == torch.int64:  # places beyond int32 stay beyond every store
            v = v.clamp(-(1 << 31), (1 << 31) - 1)
        return v.to(torch.int32).contiguous(), 0

    def _query(self, q, scale, softcap, slopes):
        self._here(q)
        if q.dim() != 3 or q.shape[0] != self.BH or q.shape[2] != self.d or q.shape[1] < 1:
            raise ValueError(f"q {tuple(q.shape)} must be [{self.BH}, G, {self.d}]")
        q = (q if q.dtype in _KDT else q.float()).contiguous()
        q = q.clone() if q.data_ptr() % 16 else q
        softcap = 0.0 if softcap is None else float(softcap)
        if not softcap >= 0.0:
            raise ValueError(f"softcap {softcap} must be positive (None or 0: no cap)")
        if slopes is not None:
            self._here(slopes)
            slopes = slopes.float().expand(q.shape[:2]).contiguous()
        return q, float(self.d) ** -0.5 if scale is None else float(scale), softcap, slopes

    def _workspace(self, nbytes):
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None

    # ------------------------------------------------------------------ writing and reading
    def write(self, K, V, pos=0):
        """Quantise K, V [BH, T, d] into tokens pos .. pos + T - 1 of each row: a
        prompt, a piece of one, or one step's token.

        A 64-token block's scale is its largest finite |x| / 448 (e4m3) or 127 (int8); a
        block that holds earlier tokens keeps its scale, or takes the least
        power-of-two multiple of it that holds the new tokens, to which its earlier
        codes are then rounded.  Tokens at pos + T and behind are no longer the row's.
        With a tensor `pos`, rows whose tokens do not all fit into the store (a negative
        pos among them) are left as they are; an int pos that does not fit raises.  K
        and V may be views with any strides (their rows dense)."""
        self._here(K, V)
        if K.dim() != 3 or K.shape != V.shape or K.shape[0] != self.BH or K.shape[2] != self.d or K.dtype != V.dtype:
            raise ValueError(f"K {K.dtype} {tuple(K.shape)} and V {V.dtype} {tuple(V.shape)} must be alike, "
                             f"[{self.BH}, T, {self.d}]")
        rows, at = self._per_row(pos, "pos")
        K, V = _aligned(K), _aligned(V)
        self._call("fathom_rows8_write", _ptr(K), _ptr(V), _KDT[K.dtype], K.stride(0), K.stride(1), V.stride(0), V.stride(1),
                   _ptr(rows), at, self.BH, K.shape[1], self.d, self.cap, self._code, *self._tensors())

    def _read(self, idx, rows, at, R, dtype):
        if dtype not in _KDT:
            raise ValueError(f"dtype {dtype} unsupported (float32, float16, bfloat16)")
        K, V = (torch.empty(self.BH, R, self.d, dtype=dtype, device=self.device) for _ in "kv")
        self._call("fathom_rows8_read", *self._tensors(), self._code, self.BH, self.cap, self.d, _ptr(idx), _ptr(rows), at, R,
                   _KDT[dtype], _ptr(K), _ptr(V))
        return K, V

    def read(self, pos, T, dtype=torch.bfloat16):
        """The values of tokens pos .. pos + T - 1 of each row, K, V [BH, T, d];
        tokens outside the store are zeros."""
        rows, at = self._per_row(pos, "pos")
        return self._read(None, rows, at, int(T), dtype)

    def gather_rows(self, idx, dtype=torch.bfloat16):
        """The values of the listed tokens idx [BH, R], K, V [BH, R, d]; tokens outside
        the store give zero rows, as offload.gather_rows does."""
        self._here(idx)
        if idx.dim() != 2 or idx.shape[0] != self.BH:
            raise ValueError(f"idx {tuple(idx.shape)} must be [{self.BH}, R]")
        return self._read(idx.to(torch.int64).contiguous(), None, 0, idx.shape[1], dtype)

    # ------------------------------------------------------------------ attention
    def attention(self, q, length, window=0, scale=None, softcap=None, slopes=None):
        """Attention of one token per row, q [BH, G, d] (float32, float16 or bfloat16),
        over the row's first `length` tokens, or the last `window` of them (0: all):
        softmax(z) . V in float32 [BH, G, d], with
          z_t = scale q . K_t, capped to softcap tanh(z_t / softcap) if softcap is given,
                then biased by slopes[bh, g] (t - (length - 1)) if slopes are given
        (slopes [BH, G], or [G]; scale defaults to d ** -0.5).  A tensor length is taken
        as within [0, cap].  A row without tokens gives zeros."""
        q, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        lens, n = self._per_row(length, "length")
        G, window = q.shape[1], int(window)
        positions = self.cap if lens is not None else n
        positions = min(positions, window) if window > 0 else positions
        nbytes = _lib.lib().fathom_rows8_attention_workspace_bytes(self.BH, G, self.d, positions)
        ws = self._workspace(nbytes)
        out = torch.empty(self.BH, G, self.d, dtype=torch.float32, device=self.device)
        self._call("fathom_rows8_attention", _ptr(q), _KDT[q.dtype], *self._tensors(), self._code, self.BH, G, self.d,
                   self.cap, _ptr(lens), n, window, scale, softcap, _ptr(slopes), _ptr(out), _ptr(ws), nbytes)
        return out

    def gather_attention(self, q, idx, length=None, scale=None, softcap=None, slopes=None):
        """The same attention over the selected tokens idx [BH, G, k] (as
        PlaneStore.scan_topk gives them): [BH, G, d] float32.  A token listed twice counts
        twice.  Tokens outside [0, length) (length defaults to cap) take no part, so a
        selection may be padded with -1 (offload.gather_attention's zero rows score 0
        instead)."""
        q, scale, softcap, slopes = self._query(q, scale, softcap, slopes)
        self._here(idx)
        G = q.shape[1]
        if idx.dim() != 3 or idx.shape[:2] != q.shape[:2]:
            raise ValueError(f"idx {tuple(idx.shape)} must be [{self.BH}, {G}, k]")
        idx = idx.to(torch.int64).contiguous()
        k = idx.shape[2]
        lens, n = self._per_row(self.cap if length is None else length, "length")
        nbytes = _lib.lib().fathom_rows8_gather_attention_workspace_bytes(self.BH, G, self.d, k)
        ws = self._workspace(nbytes)
        out = torch.empty(self.BH, G, self.d, dtype=torch.float32, device=self.device)
        self._call("fathom_rows8_gather_attention", _ptr(q), _KDT[q.dtype], _ptr(idx), *self._tensors(), self._code, self.BH,
                   G, k, self.d, self.cap, _ptr(lens), n, scale, softcap, _ptr(slopes), _ptr(out), _ptr(ws), nbytes)
        return out
