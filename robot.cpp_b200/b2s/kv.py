"""Python binding of the key/value cache operators in libb2s.so (C ABI in include/b2s_kv.h).

    cache = kv.Cache.empty(n_pages, n_kv_heads, page_size, head_dim)      # 8-bit pages and their scales
    kv.rope_axes(qk, n_heads + n_kv_heads, head_dim, pos, sections, theta, qk)
    kv.write(cache, k, v, slots)                                          # slot = page * page_size + token
    batch = kv.Batch(q_start, kv_len, pages, max_q)
    ws = torch.empty(kv.attention_workspace_size(cache, batch, q.shape[0], n_heads), dtype=torch.uint8, device="cuda")
    kv.attention(cache, batch, q, n_heads, scale, True, o, ws)

Every call only enqueues work on the given stream (default: torch's current one) of the current device. Handles keep
the tensors they describe.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import check, lib as _lib

TYPE_F32 = 0
TYPE_I8 = 24
TYPE_BF16 = 30
TYPE_F8_E4M3 = 1037

_ACT = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16}
_CODE = {torch.int8: TYPE_I8, torch.float8_e4m3fn: TYPE_F8_E4M3}


class CacheStruct(C.Structure):
    """Mirror of b2s_kv_cache."""
    _fields_ = [("type", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32),
                ("n_pages", C.c_int64), ("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p),
                ("v_scale", C.c_void_p)]


class BatchStruct(C.Structure):
    """Mirror of b2s_kv_batch."""
    _fields_ = [("batch", C.c_int32), ("max_q", C.c_int32), ("q_start", C.c_void_p), ("kv_len", C.c_void_p),
                ("pages", C.c_void_p), ("max_pages", C.c_int64), ("ld_pages", C.c_int64)]


EXPORTED = ["b2s_rope_axes", "b2s_kv_write", "b2s_kv_read", "b2s_attention_kv_workspace_size", "b2s_attention_kv",
            "b2s_attention_kv_prefix"]

_L = None


def _bind():
    global _L
    if _L is None:
        L = _lib()
        vp, i64, i32, f32, sz = C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_size_t
        sig = {
            "b2s_rope_axes": (C.c_int, [i32, vp, i64, i64, C.c_int, C.c_int, vp, i64, C.c_int, vp, C.c_int, f32, vp, i64,
                                        vp]),
            "b2s_kv_write": (C.c_int, [vp, i32, vp, i64, vp, i64, i64, vp, vp]),
            "b2s_kv_read": (C.c_int, [vp, vp, i64, i32, vp, i64, vp, i64, vp]),
            "b2s_attention_kv_workspace_size": (sz, [vp, vp, i64, C.c_int, i64]),
            "b2s_attention_kv": (C.c_int, [vp, vp, i32, vp, i64, i64, C.c_int, f32, C.c_int, vp, i64, vp, sz, vp]),
            "b2s_attention_kv_prefix": (C.c_int, [vp, vp, vp, i64, i32, vp, i64, i64, C.c_int, f32, C.c_int, vp, i64, vp,
                                                  sz, vp]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _L = L
    return _L


# ---------------------------------------------------------------------------------------------- argument checks
def _here(t, what: str):
    """The tensor is on the current device, where the library launches."""
    if not t.is_cuda or t.get_device() != torch.cuda.current_device():
        raise ValueError(f"{what} must be on the current CUDA device, it is on {t.device}")


def _rows(x, width: int, what: str, dtype=None):
    """A matrix of f32 or bf16 rows with contiguous values: (type, pointer, row stride)."""
    if x.dim() != 2 or x.shape[1] != width or x.stride(1) != 1:
        raise ValueError(f"{what} must be a matrix with rows of {width} contiguous values, got {tuple(x.shape)} with "
                         f"strides {tuple(x.stride())}")
    if x.dtype not in _ACT or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{what} has dtype {x.dtype}" + (f", not {dtype}" if dtype is not None else ", not float32 or bfloat16"))
    _here(x, what)
    # a single row may have any stride: it is never used
    return _ACT[x.dtype], x.data_ptr(), x.stride(0) if x.shape[0] > 1 else width


def _ints(t, dtype, shape, what: str) -> int:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    _here(t, what)
    return t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)


# ---------------------------------------------------------------------------------------------- handles
class Cache:
    """A paged 8-bit cache: codes [n_pages, n_kv_heads, page_size, head_dim] (int8 or float8_e4m3fn) and fp32 scales
    [n_pages, n_kv_heads, page_size], for keys and for values."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.dtype not in _CODE:
            raise ValueError(f"k must hold int8 or float8_e4m3fn codes [pages, heads, page_size, head_dim], got {k.dtype} "
                             f"{tuple(k.shape)}")
        for t, like, what in ((k, k, "k"), (v, k, "v"), (k_scale, k_scale, "k_scale"), (v_scale, v_scale, "v_scale")):
            shape = tuple(k.shape) if like is k else tuple(k.shape[:3])
            dtype = k.dtype if like is k else torch.float32
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {shape} on {k.device}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.struct = CacheStruct(_CODE[k.dtype], self.n_kv_heads, self.head_dim, self.page_size, self.n_pages, k.data_ptr(),
                                  v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self.ref = C.addressof(self.struct)
        self.width = self.n_kv_heads * self.head_dim

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, dtype=torch.int8, device="cuda"):
        """A cache of uninitialised pages."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        codes = [torch.empty(shape, dtype=dtype, device=device) for _ in range(2)]
        return cls(*codes, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


class Batch:
    """The sequences of an attention call: q_start [batch + 1], kv_len [batch] and pages [batch, max_pages], all int32;
    the tensors may be written between calls, their shapes and max_q stay."""

    def __init__(self, q_start, kv_len, pages, max_q: int):
        b = kv_len.shape[0]
        if pages.dim() != 2 or pages.shape[0] != b or pages.dtype != torch.int32 or (pages.shape[1] > 1 and pages.stride(1) != 1):
            raise ValueError(f"pages must be an int32 matrix of {b} rows, got {pages.dtype} {tuple(pages.shape)}")
        _here(pages, "pages")
        self.q_start, self.kv_len, self.pages, self.max_q = q_start, kv_len, pages, int(max_q)
        self.struct = BatchStruct(b, self.max_q, _ints(q_start, torch.int32, (b + 1,), "q_start"),
                                  _ints(kv_len, torch.int32, (b,), "kv_len"), pages.data_ptr(), pages.shape[1],
                                  pages.stride(0) if b > 1 else pages.shape[1])
        self.ref = C.addressof(self.struct)


# ---------------------------------------------------------------------------------------------- operators
def rope_axes(x, n_heads: int, head_dim: int, pos, sections, theta_base: float, y, interleaved: bool = False,
              stream=None) -> None:
    """Rotates rows of n_heads heads (NEOX pairs) by positions pos [M, axes] int32; sections[a] pairs turn by axis a, in
    blocks or dealt in turn (interleaved). y may be x."""
    width = n_heads * head_dim
    ty, px, ldx = _rows(x, width, "x")
    _, py, ldy = _rows(y, width, "y", x.dtype)
    n = len(sections)
    if y.shape[0] != x.shape[0] or px == py and x.stride(0) != y.stride(0):
        raise ValueError("x and y must have the same rows")
    pp = _ints(pos, torch.int32, (x.shape[0], n), "pos")
    check(_bind().b2s_rope_axes(ty, px, ldx, x.shape[0], n_heads, head_dim, pp, n, n, (C.c_int32 * n)(*sections),
                                int(interleaved), theta_base, py, ldy, _stream(stream)))


def write(cache: Cache, k, v, slots, stream=None) -> None:
    """Quantises rows of keys and values [M, n_kv_heads * head_dim] into slots [M] int64 (negative: skipped)."""
    ty, pk, ldk = _rows(k, cache.width, "k")
    _, pv, ldv = _rows(v, cache.width, "v", k.dtype)
    if v.shape[0] != k.shape[0]:
        raise ValueError("k and v must have the same rows")
    _here(cache.k, "cache")
    check(_bind().b2s_kv_write(cache.ref, ty, pk, ldk, pv, ldv, k.shape[0],
                               _ints(slots, torch.int64, (k.shape[0],), "slots"), _stream(stream)))


def read(cache: Cache, slots, k=None, v=None, stream=None) -> None:
    """Reads slots [M] int64 back into rows k and / or v (zeros for a negative slot)."""
    M = slots.shape[0]
    ty, pk, ldk, pv, ldv = TYPE_F32, None, 0, None, 0
    if k is not None:
        ty, pk, ldk = _rows(k, cache.width, "k")
    if v is not None:
        ty, pv, ldv = _rows(v, cache.width, "v", None if k is None else k.dtype)
    if any(t is not None and t.shape[0] != M for t in (k, v)):
        raise ValueError(f"k and v must have {M} rows")
    _here(cache.k, "cache")
    check(_bind().b2s_kv_read(cache.ref, _ints(slots, torch.int64, (M,), "slots"), M, ty, pk, ldk, pv, ldv, _stream(stream)))


def attention_workspace_size(cache: Cache, batch: Batch, M: int, n_heads: int, prefix_len: int = 0) -> int:
    """Workspace bytes of attention() (or, with prefix_len, attention_prefix()) for M query rows."""
    return int(_bind().b2s_attention_kv_workspace_size(cache.ref, batch.ref, M, n_heads, prefix_len))


def _qo(cache, q, o, n_heads, workspace):
    width = n_heads * cache.head_dim
    ty, pq, ldq = _rows(q, width, "q")
    _, po, ldo = _rows(o, width, "o", q.dtype)
    if o.shape[0] != q.shape[0]:
        raise ValueError("q and o must have the same rows")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _here(cache.k, "cache")
    _here(workspace, "workspace")
    return ty, pq, ldq, po, ldo


def attention(cache: Cache, batch: Batch, q, n_heads: int, scale: float, causal: bool, o, workspace, stream=None) -> None:
    """o = softmax(scale q K^T) V of each sequence's query rows over its cached tokens (its last tokens, if causal)."""
    ty, pq, ldq, po, ldo = _qo(cache, q, o, n_heads, workspace)
    check(_bind().b2s_attention_kv(cache.ref, batch.ref, ty, pq, ldq, q.shape[0], n_heads, scale, int(bool(causal)), po, ldo,
                                   workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(stream)))


def attention_prefix(cache: Cache, batch: Batch, prefix_pages, prefix_len: int, q, n_heads: int, scale: float,
                     causal: bool, o, workspace, stream=None) -> None:
    """attention() with prefix_len tokens in prefix_pages [pages] int32 in front of every sequence."""
    ty, pq, ldq, po, ldo = _qo(cache, q, o, n_heads, workspace)
    need = -(-prefix_len // cache.page_size)
    if prefix_pages.dim() != 1 or prefix_pages.shape[0] < need:
        raise ValueError(f"prefix_pages must hold {need} pages")
    pp = _ints(prefix_pages, torch.int32, tuple(prefix_pages.shape), "prefix_pages")
    check(_bind().b2s_attention_kv_prefix(cache.ref, batch.ref, pp, prefix_len, ty, pq, ldq, q.shape[0], n_heads, scale,
                                          int(bool(causal)), po, ldo, workspace.data_ptr(),
                                          workspace.numel() * workspace.element_size(), _stream(stream)))
