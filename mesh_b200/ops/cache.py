"""A layer's key/value cache, in bf16 or in 8-bit codes: rows written, read back, and the accepted branch of a tree kept.

The cache has the layout of the decode kernels' (``ops/decode.py``), ``[B, kv_heads, max_seq, head_dim]``.  With 8 bits a row
(one token and head) is int8 codes and one fp32 scale: with ``a = max |x|``, ``scale = a / 127`` and ``code = round(127 x / a)``,
ties to even; it stands for ``code * scale``.  A row with a NaN or an infinity gets the scale NaN.

Reference: the E2B decode analysis's KV cache (design/e2b-crossover-2026-09-16.md:42-52).
"""
from __future__ import annotations

import ctypes
from ctypes import c_char_p, c_int, c_longlong, c_void_p

import torch

from .. import _native
from ..utils.status import status_block


class _Cache(ctypes.Structure):
    """``MeshKvCache`` (csrc/ops/draft_api.h)."""
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p),
                ("B", c_int), ("kv_heads", c_int), ("max_seq", c_int), ("head_dim", c_int), ("bits", c_int)]


_I32 = torch.int32
_bound = None


def _lib() -> ctypes.CDLL:
    """The library with the signatures of this family's calls set: with them, addresses and numbers go through as they are, which
    is half of a call's host time."""
    global _bound
    if _bound is None:
        L = _native.lib()
        P, I, Q = c_void_p, c_int, c_longlong
        for name, types in (("mesh_kv_append", [P, P, P, Q, Q, Q, Q, Q, Q, P, P, I, P]), ("mesh_kv_read", [P, P, P, P, P, I, P]),
                            ("mesh_kv_keep", [P, I, P, P, P, I, P]), ("mesh_draft_attention", [P, c_char_p, P]),
                            ("mesh_constrain_logits", [c_char_p, P])):
            getattr(L, name).argtypes = types
        L.mesh_draft_attention_scratch.argtypes, L.mesh_draft_attention_scratch.restype = [P, c_char_p], Q
        _bound = L
    return _bound


def _launch(index: int, name: str, launches: int, *args) -> None:
    """Calls ``name(*args, stream)`` on the current stream of device ``index`` (-1: not a GPU)."""
    if index < 0:
        raise ValueError(f"{name}: the tensors are on the host; the kernels need a GPU")
    fn = getattr(_lib(), name)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, name)
    _native.count_launch(launches)


def _index(device: torch.device) -> int:
    return device.index if device.type == "cuda" else -1


def _ints(t: torch.Tensor | None, name: str, device: torch.device, shape: tuple) -> int:
    """Address of an int32 tensor of this shape (0 for ``None``)."""
    if t is None:
        return 0
    if t.dtype is not _I32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: need a contiguous int32 tensor of shape {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _meet(tensors) -> bool:
    """Whether two of these contiguous tensors have bytes in common."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t is not None and t.numel())
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


class KVCache:
    """Handle of one layer's cache: ``k``, ``v`` ``[B, kv_heads, max_seq, head_dim]`` in bf16, or int8 codes with ``k_scale``,
    ``v_scale`` ``[B, kv_heads, max_seq]`` in fp32.  The tensors must keep their addresses while the handle is used."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("KVCache: k and v must be [B, kv_heads, max_seq, head_dim] alike")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("KVCache: k and v must be contiguous")
        if k.shape[3] not in (64, 128, 256):
            raise ValueError(f"KVCache: head_dim must be 64, 128 or 256, got {k.shape[3]}")
        if k.dtype == torch.int8:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != k.device or not s.is_contiguous():
                    raise ValueError("KVCache: int8 codes need contiguous fp32 scales [B, kv_heads, max_seq]")
        elif k.dtype != torch.bfloat16:
            raise ValueError(f"KVCache: rows are bf16 or int8, got {k.dtype}")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("KVCache: bf16 rows have no scales")
        if k.shape[1] < 1 or k.shape[2] < 1:
            raise ValueError("KVCache: empty cache")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.bits = 8 if k.dtype == torch.int8 else 16
        B, H, S, hd = k.shape
        self._c = _Cache(k.data_ptr(), v.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
                         0 if v_scale is None else v_scale.data_ptr(), B, H, S, hd, self.bits)
        self._at, self._index = ctypes.addressof(self._c), _index(k.device)
        self._status = status_block(k.device).data_ptr() if self._index >= 0 else 0
        self._shared = _meet((k, v, k_scale, v_scale))
        self._scratch: dict = {}                 # floats of scratch by the sizes of a call (ops/draft.py)

    @classmethod
    def empty(cls, B: int, kv_heads: int, max_seq: int, head_dim: int, bits: int = 8, device="cuda") -> "KVCache":
        """A cache of zeros: bf16 rows (``bits=16``) or 8-bit ones."""
        if bits not in (8, 16):
            raise ValueError(f"KVCache: bits must be 8 or 16, got {bits}")
        dtype = torch.int8 if bits == 8 else torch.bfloat16
        k = torch.zeros((B, kv_heads, max_seq, head_dim), dtype=dtype, device=device)
        s = torch.zeros((2, B, kv_heads, max_seq), dtype=torch.float32, device=device) if bits == 8 else (None, None)
        return cls(k, torch.zeros_like(k), s[0], s[1])

    def append(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """Row ``k[b, t]``, ``v[b, t]`` (``[B, T, kv_heads, head_dim]`` bf16, any strides with a dense last dimension: columns of a fused
        projection, for instance; not rows of this cache) goes to slot ``pos[b] + t`` for ``t < counts[b]`` (int32; ``None``: all).  Rows
        outside the cache are not written."""
        B, H, S, hd = self.k.shape
        T = k.shape[1] if k.dim() == 4 else -1
        for x in (k, v):
            if x.shape != (B, T, H, hd) or x.dtype is not torch.bfloat16 or x.device != self.device:
                raise ValueError(f"append: rows must be bf16 [{B}, T, {H}, {hd}] on {self.device}, got {x.dtype} {list(x.shape)} on {x.device}")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("append: the last dimension must be dense")
        p, n = _ints(pos, "append: pos", self.device, (B,)), _ints(counts, "append: counts", self.device, (B,))
        if self._shared:
            raise ValueError("append: keys and values of this cache share memory: it can be read, not written")
        if B == 0 or T == 0:
            return
        _launch(self._index, "mesh_kv_append", 1, self._at, k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], p, n, T)

    def read(self, start: torch.Tensor, T: int, counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows ``start[b] .. start[b] + T`` as dense bf16 ``[B, T, kv_heads, head_dim]`` keys and values; zero behind ``counts[b]`` and
        outside the cache.  ``ops.attention.flash_attention`` takes them where all sequences are equally long; it has no lengths, and
        rows of zeros would take weight."""
        B, H, S, hd = self.k.shape
        if T < 0:
            raise ValueError("read: T must not be negative")
        p, n = _ints(start, "read: start", self.device, (B,)), _ints(counts, "read: counts", self.device, (B,))
        k = torch.empty(B, T, H, hd, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        if B and T:
            _launch(self._index, "mesh_kv_read", 1, self._at, k.data_ptr(), v.data_ptr(), p, n, T)
        return k, v

    def dequantize(self) -> tuple[torch.Tensor, torch.Tensor]:
        """What every slot stands for, in fp32 and plain PyTorch (oracle)."""
        if self.bits == 16:
            return self.k.float(), self.v.float()
        return self.k.float() * self.k_scale[..., None], self.v.float() * self.v_scale[..., None]


class CacheGroup:
    """The caches of a model's layers, of one geometry, moved together: each in memory of its own, keys and values too."""

    def __init__(self, caches: list[KVCache]):
        if not caches:
            raise ValueError("CacheGroup: no caches")
        c0 = caches[0]
        for c in caches:
            if c.k.shape != c0.k.shape or c.bits != c0.bits or c.device != c0.device:
                raise ValueError("CacheGroup: the caches must have one shape, type and device")
        if _meet([t for c in caches for t in (c.k, c.v, c.k_scale, c.v_scale)]):
            raise ValueError("CacheGroup: the caches must not share memory: rows moved twice would be wrong ones")
        self.caches, self.device = list(caches), c0.device
        self._arr = (_Cache * len(caches))(*[c._c for c in caches])
        self._at, self._index = ctypes.addressof(self._arr), c0._index

    def keep(self, pos: torch.Tensor, path: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """In every cache, slot ``pos[b] + i`` gets what slot ``pos[b] + path[b, i]`` held before the call, for ``i <
        counts[b]`` (``path`` int32 ``[B, N]``, N <= 64): the rows of the accepted nodes of a tree go to the front.  An entry whose slots do
        not both lie in the cache, or with ``path < 0``, is left out."""
        B = self.caches[0].k.shape[0]
        N = path.shape[1] if path.dim() == 2 else -1
        if N > 64:
            raise ValueError(f"keep: at most 64 rows per sequence, got {N}")
        q = _ints(path, "keep: path", self.device, (B, N))
        p, n = _ints(pos, "keep: pos", self.device, (B,)), _ints(counts, "keep: counts", self.device, (B,))
        if B == 0 or N == 0:
            return
        L = len(self.caches)
        _launch(self._index, "mesh_kv_keep", -(-L // 64), self._at, L, p, q, n, N)
