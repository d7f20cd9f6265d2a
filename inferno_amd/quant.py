"""Torch-facing helpers over the C-ABI of weights in 8 bits and of a paged key-value cache in 4 bits.

As in ``paged``: the C-ABI validates shapes, strides and sizes on the host and a non-zero status
raises InfernoError; launches go to torch's current stream on the tensors' device, or to
``stream``.  What the C-ABI cannot see (dtypes, devices, layouts) is checked here.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import INF_BF16, INF_F32, PagedKV4Struct, Strides, default_scale, lib
from .ops import _check
from .paged import PagedKV, _bytes, _current_device, _elsewhere, _on, _raw_stream, _size

_DT = {torch.float32: INF_F32, torch.bfloat16: INF_BF16}


def _float(t, name):
    """The C-ABI's type of a float32 or bfloat16 tensor."""
    dt = _DT.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name}: float32 or bfloat16 expected, got {t.dtype}")
    return dt


@functools.lru_cache(maxsize=4096)
def _strides(s):
    """inf_strides of a 4-D view's strides; the calls take it by value."""
    return Strides(*s)


# Checks of a call's tensors cost as much as its launch where they are made one by one: these take a
# device's number and give back what the call needs.


def _away(index, device, stream):
    """Whether a call on tensors of this device has to make another device or stream current first."""
    return (stream is not None or index < 0 or index != _current_device()) and _elsewhere(device, stream)


def _space(ws, nbytes, index, device):
    """(tensor, pointer, bytes) of the workspace: the caller's, else a new one of nbytes() bytes."""
    if ws is None:
        n = nbytes()
        if not n:
            return None, None, 0
        ws = torch.empty(n, dtype=torch.uint8, device=device)
    elif ws.get_device() != index or not ws.is_contiguous():
        raise ValueError(f"workspace: a dense tensor on {device} expected")
    return ws, ws.data_ptr() or None, ws.nbytes


def _matrix(t, name, index):
    """(pointer, row stride, rows, columns) of a matrix on this device with adjacent elements in a row."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name}: a matrix expected, got {len(shape)} dimensions")
    rows, cols = shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name}: a matrix with adjacent elements in a row expected")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, the others on device {index}")
    return t.data_ptr(), ld if rows > 1 or ld > cols else cols, rows, cols


def _matrix_i8(t, name, index):
    if t.dtype is not torch.int8:
        raise TypeError(f"{name}: int8 expected, got {t.dtype}")
    return _matrix(t, name, index)


def _vector(t, name, dtype, index, n):
    """The pointer of n dense elements of this type on this device (None stays None)."""
    if t is None:
        return None
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {dtype} expected, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, the others on device {index}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: {n} dense elements expected, got {tuple(t.shape)}")
    return t.data_ptr()


def _rows16(n, cols, device):
    """int8 [n, cols] whose rows lie on 16 bytes."""
    return torch.empty((n, -(-cols // 16) * 16), dtype=torch.int8, device=device)[:, :cols]


def quantize_i8(x, transpose=False, stream=None):
    """(q, scale): the rows of x [rows, cols] in 8 bits, q int8 [rows, cols] (rows on 16 bytes) and scale float32
    [rows]; with ``transpose`` its columns, q [cols, rows] and scale [cols] (weights [in, out])."""
    dev, index = x.device, x.get_device()
    dt = _float(x, "quantize_i8: x")
    ptr, ld, rows, cols = _matrix(x, "quantize_i8: x", index)
    if _away(index, dev, stream):
        with _on(dev, stream):
            return quantize_i8(x, transpose)
    n, k = (cols, rows) if transpose else (rows, cols)
    q = _rows16(n, k, dev)
    scale = torch.empty(n, dtype=torch.float32, device=dev)
    st = lib().inf_quantize_i8(ptr, ld, rows, cols, int(bool(transpose)), q.data_ptr(), -(-k // 16) * 16,
                               scale.data_ptr(), dt, _raw_stream(index))
    _check(st, "inf_quantize_i8")
    return q, scale


@functools.lru_cache(maxsize=4096)
def _product_bytes(call, M, N, K):
    return _size(getattr(lib(), call), M, N, K)


def gemm_i8_workspace(M, N, K, device="cuda"):
    """A workspace for gemm_i8 of these sizes, or of fewer rows."""
    return torch.empty(_product_bytes("inf_gemm_i8_workspace", M, N, K), dtype=torch.uint8, device=device)


def linear_i8_workspace(M, N, K, device="cuda"):
    """A workspace for linear_i8 of these sizes, or of fewer rows."""
    return torch.empty(_product_bytes("inf_linear_i8_workspace", M, N, K), dtype=torch.uint8, device=device)


def _result(out, name, shape, dtype, like, index):
    """(tensor, pointer, row stride) of a result, a new one beside `like` where none is given."""
    if out is None:
        out = like.new_empty(shape, dtype=dtype)
        return out, out.data_ptr(), shape[1]
    if out.shape != shape or out.dtype is not dtype:
        raise ValueError(f"{name}: {list(shape)} of {dtype} expected, got {list(out.shape)} of {out.dtype}")
    return out, *_matrix(out, name, index)[:2]


def gemm_i8(x, x_scale, w, w_scale, bias=None, dtype=torch.float32, out=None, workspace=None, stream=None):
    """y [M, N] = x w^T times the scales of x's rows and w's rows, plus bias: x [M, K] and w [N, K] int8 with rows on
    16 bytes (quantize_i8's); y and bias of ``dtype``, float32 or bfloat16."""
    dev, index = x.device, x.get_device()
    px, ldx, M, K = _matrix_i8(x, "gemm_i8: x", index)
    pw, ldw, N, Kw = _matrix_i8(w, "gemm_i8: w", index)
    if K != Kw:
        raise ValueError(f"gemm_i8: x [M, K] and w [N, K] expected, got {tuple(x.shape)} and {tuple(w.shape)}")
    dtype = out.dtype if out is not None else dtype
    if dtype not in _DT:
        raise TypeError(f"gemm_i8: float32 or bfloat16 expected, got {dtype}")
    psx = _vector(x_scale, "gemm_i8: x_scale", torch.float32, index, M)
    psw = _vector(w_scale, "gemm_i8: w_scale", torch.float32, index, N)
    pb = _vector(bias, "gemm_i8: bias", dtype, index, N)
    if _away(index, dev, stream):
        with _on(dev, stream):
            return gemm_i8(x, x_scale, w, w_scale, bias, dtype, out, workspace)
    y, py, ldy = _result(out, "gemm_i8: out", (M, N), dtype, x, index)
    if M == 0:
        return y
    ws, ptr, n = _space(workspace, lambda: _product_bytes("inf_gemm_i8_workspace", M, N, K), index, dev)
    st = lib().inf_gemm_i8(M, N, K, px, ldx, psx, pw, ldw, psw, pb, py, ldy, _DT[dtype], ptr, n, _raw_stream(index))
    _check(st, "inf_gemm_i8")
    return y


def linear_i8(x, w, w_scale, bias=None, out=None, workspace=None, stream=None):
    """y [M, N] = x w^T + bias with the weights in 8 bits (w int8 [N, K], w_scale [N]: quantize_i8's, with
    ``transpose`` where they are held [in, out]); x [M, K] is taken in 8 bits row by row, y and bias have its type."""
    dev, index = x.device, x.get_device()
    dt = _float(x, "linear_i8: x")
    px, ldx, M, K = _matrix(x, "linear_i8: x", index)
    pw, ldw, N, Kw = _matrix_i8(w, "linear_i8: w", index)
    if K != Kw:
        raise ValueError(f"linear_i8: x [M, K] and w [N, K] expected, got {tuple(x.shape)} and {tuple(w.shape)}")
    psw = _vector(w_scale, "linear_i8: w_scale", torch.float32, index, N)
    pb = _vector(bias, "linear_i8: bias", x.dtype, index, N)
    if _away(index, dev, stream):
        with _on(dev, stream):
            return linear_i8(x, w, w_scale, bias, out, workspace)
    y, py, ldy = _result(out, "linear_i8: out", (M, N), x.dtype, x, index)
    if M == 0:
        return y
    ws, ptr, n = _space(workspace, lambda: _product_bytes("inf_linear_i8_workspace", M, N, K), index, dev)
    st = lib().inf_linear_i8(M, N, K, px, ldx, pw, ldw, psw, pb, py, ldy, dt, ptr, n, _raw_stream(index))
    _check(st, "inf_linear_i8")
    return y


class PagedKV4:
    """A paged key-value cache in 4 bits: pools k, v uint8 [pages, heads, page size, D / 2] (any strides with dense
    rows) and k_scale, v_scale uint8 [pages, heads, D / 32, page size] (neighbouring slots adjacent), ``table`` int32
    [rows, pages per row] and ``lens`` int32 [rows], all on one device.  The handle keeps the tensors; their
    contents may change at any time, and ``table`` and ``lens`` may be set to other tensors of the same shape."""

    def __init__(self, k, v, k_scale, v_scale, table, lens):
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("PagedKV4: k and v of one shape [pages, heads, page size, D / 2] expected")
        pages, heads, page_size, half = k.shape
        if k_scale.shape != v_scale.shape or k_scale.shape != (pages, heads, half // 16, page_size) or half % 16:
            raise ValueError("PagedKV4: k_scale and v_scale [pages, heads, D / 32, page size] expected")
        if any(t.dtype != torch.uint8 for t in (k, v, k_scale, v_scale)):
            raise TypeError("PagedKV4: uint8 pools and scales expected")
        if table.dim() != 2 or lens.dim() != 1 or table.shape[0] != lens.shape[0]:
            raise ValueError("PagedKV4: table [rows, pages] and lens [rows] expected")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("PagedKV4: the entries of a row's table must be adjacent")
        if table.dtype != torch.int32 or lens.dtype != torch.int32:
            raise TypeError("PagedKV4: table and lens must be int32")
        if not lens.is_contiguous():
            raise ValueError("PagedKV4: lens: a dense tensor expected")
        if any(t.device != k.device for t in (v, k_scale, v_scale, table, lens)):
            raise ValueError("PagedKV4: all tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale, self._table, self._lens = k, v, k_scale, v_scale, table, lens
        self.device, self.index = k.device, k.get_device()
        self.rows, self.heads, self.D, self.page_size = table.shape[0], heads, 2 * half, page_size
        self.capacity = table.shape[1] * page_size
        self.struct = PagedKV4Struct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                     *(Strides(*t.stride()) for t in (k, v, k_scale, v_scale)), table.data_ptr(),
                                     lens.data_ptr(), PagedKV._row_stride(table), self.rows, heads, self.D, page_size,
                                     table.shape[1], pages)
        self.ref = ctypes.byref(self.struct)
        self.scale = default_scale(self.D)
        self.sizes = {}  # workspace bytes by call and arguments

    @staticmethod
    def empty(pages, heads, page_size, D, table, lens):
        """A cache of new pools on the table's device."""
        if D % 32:
            raise ValueError("PagedKV4: D must be a multiple of 32")
        k, v = (torch.empty((pages, heads, page_size, D // 2), dtype=torch.uint8, device=table.device) for _ in range(2))
        ks, vs = (torch.empty((pages, heads, D // 32, page_size), dtype=torch.uint8, device=table.device)
                  for _ in range(2))
        return PagedKV4(k, v, ks, vs, table, lens)

    table = PagedKV.table
    lens = PagedKV.lens
    _row_stride = staticmethod(PagedKV._row_stride)


def _tokens(t, name, cache, T):
    """(pointer, strides) of [rows, heads, T, D] of the cache's sizes and device."""
    if t.shape != (cache.rows, cache.heads, T, cache.D):
        raise ValueError(f"{name}: [{cache.rows}, {cache.heads}, {T}, {cache.D}] expected, got {list(t.shape)}")
    if t.get_device() != cache.index:
        raise ValueError(f"{name}: on {t.device}, the cache on {cache.device}")
    return t.data_ptr(), _strides(t.stride())


def kv4_append(cache, k, v, counts=None, stream=None):
    """Writes k, v [rows, heads, T, D] (float32 or bfloat16) as the rows' last positions (``cache.lens`` counts them
    already); ``counts`` int32 [rows]: how many of the T tokens a row has."""
    dt = _float(k, "kv4_append: k")
    if k.dim() != 4 or v.dtype != k.dtype:
        raise ValueError("kv4_append: k and v [rows, heads, T, D] of one type expected")
    T = k.shape[2]
    pk, sk = _tokens(k, "kv4_append: k", cache, T)
    pv, sv = _tokens(v, "kv4_append: v", cache, T)
    pc = _vector(counts, "counts", torch.int32, cache.index, cache.rows)
    if _away(cache.index, cache.device, stream):
        with _on(cache.device, stream):
            return kv4_append(cache, k, v, counts)
    st = lib().inf_kv4_append(cache.ref, pk, sk, pv, sv, pc, T, dt, _raw_stream(cache.index))
    _check(st, "inf_kv4_append")


def kv4_read(cache, T, first=None, dtype=torch.float32, k_out=None, v_out=None, stream=None):
    """(k, v) [rows, heads, T, D]: positions first[row] + t of every row (``first`` int32 [rows], 0 by default),
    zeros outside a row's positions."""
    T = int(T)
    if (k_out is None) != (v_out is None):
        raise ValueError("kv4_read: k_out and v_out go together")
    if k_out is not None:
        dtype = k_out.dtype
        if v_out.dtype != dtype:
            raise TypeError("kv4_read: k_out and v_out of one type expected")
    dt = _DT.get(dtype)
    if dt is None:
        raise TypeError(f"kv4_read: float32 or bfloat16 expected, got {dtype}")
    pf = _vector(first, "first", torch.int32, cache.index, cache.rows)
    if _away(cache.index, cache.device, stream):
        with _on(cache.device, stream):
            return kv4_read(cache, T, first, dtype, k_out, v_out)
    if k_out is None:
        k_out = cache.k.new_empty((cache.rows, cache.heads, max(T, 0), cache.D), dtype=dtype)
        v_out = torch.empty_like(k_out)
        pk, pv = k_out.data_ptr(), v_out.data_ptr()
        sk = sv = _strides(k_out.stride())
    else:
        pk, sk = _tokens(k_out, "kv4_read: k_out", cache, T)
        pv, sv = _tokens(v_out, "kv4_read: v_out", cache, T)
    st = lib().inf_kv4_read(cache.ref, pf, T, pk, sk, pv, sv, dt, _raw_stream(cache.index))
    _check(st, "inf_kv4_read")
    return k_out, v_out


def _decode_bytes(cache, q_heads, max_len):
    return _bytes(cache, "inf_attn_decode_kv4_workspace", q_heads, max_len)


def attn_decode_kv4_workspace(cache, q_heads, max_len=None):
    """A workspace for attn_decode_kv4 with these arguments, or a shorter max_len."""
    n = _decode_bytes(cache, q_heads, cache.capacity if max_len is None else max_len)
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def attn_decode_kv4(q, cache, scale=None, max_len=None, out=None, workspace=None, stream=None):
    """Attention of one new token per row, q [rows, q_heads, 1, D] (float32 or bfloat16), over the row's
    ``cache.lens`` positions.  ``max_len`` bounds the lengths (the capacity by default)."""
    shape = q.shape
    if len(shape) != 4 or shape[0] != cache.rows or shape[2] != 1 or shape[3] != cache.D:
        raise ValueError("attn_decode_kv4: q [rows, q_heads, 1, D] of the cache's rows and D expected")
    dt = _float(q, "attn_decode_kv4: q")
    if q.get_device() != cache.index:
        raise ValueError(f"attn_decode_kv4: q must be on {cache.device}")
    heads = shape[1]
    max_len = cache.capacity if max_len is None else int(max_len)
    if _away(cache.index, cache.device, stream):
        with _on(cache.device, stream):
            return attn_decode_kv4(q, cache, scale, max_len, out, workspace)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != q.dtype or out.get_device() != cache.index:
        raise ValueError("attn_decode_kv4: out must be like q")
    ws, ptr, n = _space(workspace, lambda: _decode_bytes(cache, heads, max_len), cache.index, cache.device)
    st = lib().inf_attn_decode_kv4(cache.ref, q.data_ptr(), _strides(q.stride()), out.data_ptr(),
                                   _strides(out.stride()), heads, max_len,
                                   cache.scale if scale is None else float(scale), dt, ptr, n,
                                   _raw_stream(cache.index))
    _check(st, "inf_attn_decode_kv4")
    return out


__all__ = ["PagedKV4", "kv4_append", "kv4_read", "attn_decode_kv4", "attn_decode_kv4_workspace", "quantize_i8",
           "gemm_i8", "gemm_i8_workspace", "linear_i8", "linear_i8_workspace"]
