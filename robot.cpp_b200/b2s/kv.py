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
# A call costs the host a few microseconds, most of them here: each attribute of a tensor is read once.
_device = torch.cuda.current_device  # the device that the library launches on
# The current stream's handle; a Stream object around it takes 1.3 of a call's 8 us.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _refuse_rows(x, width: int, what: str, like, dev: int):
    if x.get_device() != dev:
        raise ValueError(f"{what} must be on the current CUDA device, it is on {x.device}")
    if x.dim() != 2 or x.shape[1] != width or x.stride(1) != 1:
        raise ValueError(f"{what} must be a matrix with rows of {width} contiguous values, got {tuple(x.shape)} with "
                         f"strides {tuple(x.stride())}")
    raise ValueError(f"{what} has dtype {x.dtype}" + (", not float32 or bfloat16" if like is None else ", unlike the others"))


def _rows(x, width: int, what: str, dev: int, like=None):
    """A matrix of f32 or bf16 rows with contiguous values: (type, rows, pointer, row stride). `like`: the type it must have."""
    shape, stride, ty = x.shape, x.stride(), _ACT.get(x.dtype)
    if len(shape) != 2 or shape[1] != width or stride[1] != 1 or ty is None or (like is not None and ty != like) or \
            x.get_device() != dev:
        _refuse_rows(x, width, what, like, dev)
    # a single row may have any stride: it is never used
    return ty, shape[0], x.data_ptr(), stride[0] if shape[0] > 1 else width


def _ints(t, dtype, shape, what: str, dev: int) -> int:
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on the current CUDA device, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _stream(stream, dev: int) -> int:
    if stream is None:
        return _raw_stream(dev)
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
        self.device = k.get_device()

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
        dev = _device()
        if pages.get_device() != dev:
            raise ValueError(f"pages must be on the current CUDA device, it is on {pages.device}")
        self.q_start, self.kv_len, self.pages, self.max_q, self.device = q_start, kv_len, pages, int(max_q), dev
        self.struct = BatchStruct(b, self.max_q, _ints(q_start, torch.int32, (b + 1,), "q_start", dev),
                                  _ints(kv_len, torch.int32, (b,), "kv_len", dev), pages.data_ptr(), pages.shape[1],
                                  pages.stride(0) if b > 1 else pages.shape[1])
        self.ref = C.addressof(self.struct)


# ---------------------------------------------------------------------------------------------- operators
def rope_axes(x, n_heads: int, head_dim: int, pos, sections, theta_base: float, y, interleaved: bool = False,
              stream=None) -> None:
    """Rotates rows of n_heads heads (NEOX pairs) by positions pos [M, axes] int32; sections[a] pairs turn by axis a, in
    blocks or dealt in turn (interleaved). y may be x."""
    width, dev = n_heads * head_dim, _device()
    ty, M, px, ldx = _rows(x, width, "x", dev)
    _, My, py, ldy = _rows(y, width, "y", dev, ty)
    n = len(sections)
    if My != M or px == py and ldx != ldy:
        raise ValueError("x and y must have the same rows")
    pp = _ints(pos, torch.int32, (M, n), "pos", dev)
    check(_bind().b2s_rope_axes(ty, px, ldx, M, n_heads, head_dim, pp, n, n, (C.c_int32 * n)(*sections), int(interleaved),
                                theta_base, py, ldy, _stream(stream, dev)))


def write(cache: Cache, k, v, slots, stream=None) -> None:
    """Quantises rows of keys and values [M, n_kv_heads * head_dim] into slots [M] int64 (negative: skipped)."""
    dev = _device()
    ty, M, pk, ldk = _rows(k, cache.width, "k", dev)
    _, Mv, pv, ldv = _rows(v, cache.width, "v", dev, ty)
    if Mv != M or cache.device != dev:
        raise ValueError("k, v and the cache must have the same rows and device")
    check(_bind().b2s_kv_write(cache.ref, ty, pk, ldk, pv, ldv, M, _ints(slots, torch.int64, (M,), "slots", dev),
                               _stream(stream, dev)))


def read(cache: Cache, slots, k=None, v=None, stream=None) -> None:
    """Reads slots [M] int64 back into rows k and / or v (zeros for a negative slot)."""
    dev = _device()
    ty, M, pk, ldk, pv, ldv = None, slots.shape[0], None, 0, None, 0
    Mk = Mv = M
    if k is not None:
        ty, Mk, pk, ldk = _rows(k, cache.width, "k", dev)
    if v is not None:
        ty, Mv, pv, ldv = _rows(v, cache.width, "v", dev, ty)
    if Mk != M or Mv != M or cache.device != dev:
        raise ValueError(f"k and v must have {M} rows and the cache's device")
    check(_bind().b2s_kv_read(cache.ref, _ints(slots, torch.int64, (M,), "slots", dev), M, TYPE_F32 if ty is None else ty, pk,
                              ldk, pv, ldv, _stream(stream, dev)))


def attention_workspace_size(cache: Cache, batch: Batch, M: int, n_heads: int, prefix_len: int = 0) -> int:
    """Workspace bytes of attention() (or, with prefix_len, attention_prefix()) for M query rows."""
    return int(_bind().b2s_attention_kv_workspace_size(cache.ref, batch.ref, M, n_heads, prefix_len))


def _qo(cache, batch, q, o, n_heads, workspace, dev):
    width = n_heads * cache.head_dim
    ty, M, pq, ldq = _rows(q, width, "q", dev)
    _, Mo, po, ldo = _rows(o, width, "o", dev, ty)
    if Mo != M:
        raise ValueError("q and o must have the same rows")
    if cache.device != dev or batch.device != dev or workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("the cache, the batch and a contiguous workspace must be on the current CUDA device")
    return ty, M, pq, ldq, po, ldo


def attention(cache: Cache, batch: Batch, q, n_heads: int, scale: float, causal: bool, o, workspace, stream=None) -> None:
    """o = softmax(scale q K^T) V of each sequence's query rows over its cached tokens (its last tokens, if causal)."""
    dev = _device()
    ty, M, pq, ldq, po, ldo = _qo(cache, batch, q, o, n_heads, workspace, dev)
    check(_bind().b2s_attention_kv(cache.ref, batch.ref, ty, pq, ldq, M, n_heads, scale, int(bool(causal)), po, ldo,
                                   workspace.data_ptr(), workspace.nbytes, _stream(stream, dev)))


def attention_prefix(cache: Cache, batch: Batch, prefix_pages, prefix_len: int, q, n_heads: int, scale: float,
                     causal: bool, o, workspace, stream=None) -> None:
    """attention() with prefix_len tokens in prefix_pages [pages] int32 in front of every sequence."""
    dev = _device()
    ty, M, pq, ldq, po, ldo = _qo(cache, batch, q, o, n_heads, workspace, dev)
    if prefix_pages.dim() != 1 or prefix_pages.shape[0] * cache.page_size < prefix_len:
        raise ValueError(f"prefix_pages must hold the pages of {prefix_len} tokens")
    pp = _ints(prefix_pages, torch.int32, prefix_pages.shape, "prefix_pages", dev)
    check(_bind().b2s_attention_kv_prefix(cache.ref, batch.ref, pp, prefix_len, ty, pq, ldq, M, n_heads, scale,
                                          int(bool(causal)), po, ldo, workspace.data_ptr(), workspace.nbytes,
                                          _stream(stream, dev)))
