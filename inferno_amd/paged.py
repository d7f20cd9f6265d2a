"""Torch-facing helpers over the C-ABI of generation from a paged key-value cache.

As in ``ops``: the C-ABI validates shapes, strides and sizes on the host and a non-zero status
raises InfernoError; launches go to torch's current stream on the tensors' device, or to
``stream``.  What the C-ABI cannot see (dtypes, devices, dense layouts) is checked here.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import InfernoError, PagedKVStruct, Strides, default_scale, lib
from .ops import _check, _dt, strides_of


# the current stream's handle on a device; the public spelling costs as much as a launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
# likewise the current device's number (asked of tensors on the GPU only: it is initialised)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


@contextlib.contextmanager
def _on(device, stream):
    """The device, and the stream where one is given, made current: new tensors belong to it."""
    if stream is not None and not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _elsewhere(device, stream):
    """Whether a call on tensors of this device has to make another device or stream current first."""
    if device.type != "cuda":
        raise ValueError(f"tensors on the GPU expected, got {device}")
    return stream is not None or device.index != _current_device()


def _of(t, name, dtype, device, shape=None):
    """A dense tensor of this dtype, device and shape, as a pointer (None stays None)."""
    if t is None:
        return None
    if t.dtype != dtype:
        raise TypeError(f"{name}: {dtype} expected, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, the others on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: a dense tensor expected")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(shape)} expected, got {tuple(t.shape)}")
    return t.data_ptr()


def _size(call, *args) -> int:
    out = ctypes.c_size_t(0)
    _check(call(*args, ctypes.byref(out)), call.__name__)
    return int(out.value)


def _workspace(ws, nbytes, device):
    """(tensor, pointer, bytes) of the workspace: the caller's, else a new one of nbytes() bytes."""
    if ws is None:
        ws = torch.empty(nbytes(), dtype=torch.uint8, device=device)
    elif ws.device != device or not ws.is_contiguous():
        raise ValueError(f"workspace: a dense tensor on {device} expected")
    return ws, ws.data_ptr() or None, ws.nbytes


class PagedKV:
    """A paged key-value cache: pools k, v [pages, heads, page size, D] (any strides with dense
    rows; with a leading layer axis, see ``layer``), ``table`` int32 [rows, pages per row] and
    ``lens`` int32 [rows], all on one device.  The handle keeps the tensors; their contents may
    change at any time, and ``table`` and ``lens`` may be set to other tensors of the same shape."""

    def __init__(self, k, v, table, lens):
        if k.shape != v.shape or k.dim() not in (4, 5):
            raise ValueError("PagedKV: k and v of one shape [pages, heads, page size, D], or [layers, ...] expected")
        if k.dtype != v.dtype or k.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"PagedKV: float32 or bfloat16 pools of one type expected, got {k.dtype} and {v.dtype}")
        if table.dim() != 2 or lens.dim() != 1 or table.shape[0] != lens.shape[0]:
            raise ValueError("PagedKV: table [rows, pages] and lens [rows] expected")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("PagedKV: the entries of a row's table must be adjacent")
        if table.dtype != torch.int32 or lens.dtype != torch.int32:
            raise TypeError("PagedKV: table and lens must be int32")
        if not (k.device == v.device == table.device == lens.device):
            raise ValueError("PagedKV: k, v, table and lens must be on one device")
        self.k, self.v, self._table, self._lens = k, v, table, lens
        self.device, self.dtype = k.device, k.dtype
        self.layers = k.shape[0] if k.dim() == 5 else 1
        self.layer_strides = (k.stride(0), v.stride(0)) if k.dim() == 5 else (0, 0)
        pages, heads, page_size, D = k.shape[-4:]
        self.rows, self.heads, self.D, self.page_size = table.shape[0], heads, D, page_size
        self.capacity = table.shape[1] * page_size
        sk, sv = (Strides(*t.stride()[-4:]) for t in (k, v))
        self.struct = PagedKVStruct(k.data_ptr(), v.data_ptr(), sk, sv, table.data_ptr(), lens.data_ptr(),
                                    self._row_stride(table), self.rows, heads, D, page_size, table.shape[1], pages,
                                    _dt(k))
        self.ref = ctypes.byref(self.struct)
        self.meta_shape = (self.rows, heads, self.capacity)
        self.scale = default_scale(D)
        self.sizes = {}  # workspace bytes by call and arguments

    @staticmethod
    def _row_stride(table):
        return table.stride(0) if table.shape[0] > 1 else max(table.stride(0), table.shape[1])

    @property
    def table(self):
        return self._table

    @table.setter
    def table(self, t):
        if (t.shape != self._table.shape or t.dtype != torch.int32 or t.device != self.device
                or (t.shape[1] > 1 and t.stride(1) != 1)):
            raise ValueError("PagedKV: an int32 table of the same shape and device expected")
        self._table = t
        self.struct.table, self.struct.table_stride = t.data_ptr(), self._row_stride(t)

    @property
    def lens(self):
        return self._lens

    @lens.setter
    def lens(self, t):
        _of(t, "lens", torch.int32, self.device, self._lens.shape)
        self._lens = t
        self.struct.lens = t.data_ptr()

    def layer(self, i):
        """The cache of layer i of pools with a layer axis; it has the table and lens of now."""
        if self.k.dim() != 5:
            raise ValueError("PagedKV.layer: the pools have no layer axis")
        return PagedKV(self.k[i], self.v[i], self._table, self._lens)

    def meta(self, dtype):
        """Zeros [rows, heads, capacity]: room for the weights (float32) or positions (int32)."""
        return torch.zeros(self.meta_shape, dtype=dtype, device=self.device)


def _one_layer(cache, what):
    if cache.k.dim() != 4:
        raise ValueError(f"{what}: the cache of one layer expected (PagedKV.layer)")


def _bytes(cache, call, *args):
    """The workspace bytes that the C-ABI's `call` gives, asked once per cache and arguments (a bounded number of them:
    ``max_len`` may be another one at every token)."""
    n = cache.sizes.get((call, args))
    if n is None:
        if len(cache.sizes) >= 4096:
            cache.sizes.clear()
        n = cache.sizes[call, args] = _size(getattr(lib(), call), cache.ref, *args)
    return n


def kv_append(cache, k, v, counts=None, weights=None, positions=None, seen=None, stream=None):
    """Writes k, v [rows, heads, T, D] as the rows' last positions (``cache.lens`` counts them
    already); ``counts`` int32 [rows]: how many of the T tokens a row has.  ``weights`` float32
    and ``positions`` int32 [rows, heads, capacity] are set for the new tokens."""
    dev = cache.device
    _one_layer(cache, "kv_append")
    shape = k.shape
    if v.shape != shape or len(shape) != 4 or shape[0] != cache.rows or shape[1] != cache.heads or shape[3] != cache.D:
        raise ValueError("kv_append: k and v [rows, heads, T, D] of the cache's rows, heads and D expected")
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise TypeError("kv_append: k and v must have the cache's dtype")
    if k.device != dev or v.device != dev:
        raise ValueError(f"kv_append: k and v must be on {dev}")
    rows = (cache.rows,)
    pc, ps = _of(counts, "counts", torch.int32, dev, rows), _of(seen, "seen", torch.int32, dev, rows)
    pw = _of(weights, "weights", torch.float32, dev, cache.meta_shape)
    pp = _of(positions, "positions", torch.int32, dev, cache.meta_shape)
    if _elsewhere(dev, stream):
        with _on(dev, stream):
            return kv_append(cache, k, v, counts, weights, positions, seen)
    st = lib().inf_kv_append(cache.ref, k.data_ptr(), strides_of(k), v.data_ptr(), strides_of(v), pc, shape[2], pw, pp,
                             ps, _raw_stream(dev.index))
    _check(st, "inf_kv_append")


def _decode_bytes(cache, q_heads, max_len, weights):
    return _bytes(cache, "inf_attn_decode_paged_workspace", q_heads, max_len, int(bool(weights)))


def attn_decode_paged_workspace(cache, q_heads, max_len=None, weights=False):
    """A workspace for attn_decode_paged with these arguments."""
    n = _decode_bytes(cache, q_heads, cache.capacity if max_len is None else max_len, weights)
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def attn_decode_paged(q, cache, scale=None, max_len=None, weights=None, weights_out=None, out=None, workspace=None,
                      stream=None):
    """Attention of one new token per row, q [rows, q_heads, 1, D], over the row's ``cache.lens``
    positions.  ``max_len`` bounds the lengths (the capacity by default).  ``weights_out`` (float32
    [rows, heads, capacity]) gets ``weights`` (zeros if None, may be the same tensor) plus every position's
    probabilities, summed over the query heads of its head."""
    dev = cache.device
    _one_layer(cache, "attn_decode_paged")
    shape = q.shape
    if len(shape) != 4 or shape[0] != cache.rows or shape[2] != 1 or shape[3] != cache.D:
        raise ValueError("attn_decode_paged: q [rows, q_heads, 1, D] of the cache's rows and D expected")
    if q.dtype != cache.dtype or q.device != dev:
        raise ValueError(f"attn_decode_paged: q must be {cache.dtype} on {dev}")
    if weights is not None and weights_out is None:
        raise ValueError("attn_decode_paged: weights without weights_out")
    heads = shape[1]
    max_len = cache.capacity if max_len is None else int(max_len)
    w_in = _of(weights, "weights", torch.float32, dev, cache.meta_shape)
    w_out = _of(weights_out, "weights_out", torch.float32, dev, cache.meta_shape)
    if _elsewhere(dev, stream):
        with _on(dev, stream):
            return attn_decode_paged(q, cache, scale, max_len, weights, weights_out, out, workspace)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != q.dtype or out.device != dev:
        raise ValueError("attn_decode_paged: out must be like q")
    ws, ptr, n = _workspace(workspace, lambda: _decode_bytes(cache, heads, max_len, w_out), dev)
    st = lib().inf_attn_decode_paged(cache.ref, q.data_ptr(), strides_of(q), out.data_ptr(), strides_of(out), heads,
                                     max_len, cache.scale if scale is None else float(scale), w_in, w_out, ptr, n,
                                     _raw_stream(dev.index))
    _check(st, "inf_attn_decode_paged")
    return out


def _evict_bytes(cache, keep, max_len):
    return _bytes(cache, "inf_kv_evict_workspace", keep, max_len)


def kv_evict_workspace(cache, keep, max_len=None):
    """A workspace for kv_evict with these arguments."""
    n = _evict_bytes(cache, keep, cache.capacity if max_len is None else max_len)
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def kv_evict(cache, weights, positions, keep, recent=0, weights_out=None, positions_out=None, lens_out=None,
             max_len=None, workspace=None, stream=None):
    """Cuts every row and head to its ``keep`` positions of the largest weights, the ``recent`` newest
    among them, in place in the pools.  ``weights_out`` and ``positions_out`` are the inputs
    by default; returns the new lengths (``lens_out``, which may be ``cache.lens``)."""
    dev = cache.device
    _one_layer(cache, "kv_evict")
    keep, meta = int(keep), cache.meta_shape
    max_len = cache.capacity if max_len is None else int(max_len)
    pw, pp = _of(weights, "weights", torch.float32, dev, meta), _of(positions, "positions", torch.int32, dev, meta)
    if _elsewhere(dev, stream):
        with _on(dev, stream):
            return kv_evict(cache, weights, positions, keep, recent, weights_out, positions_out, lens_out, max_len,
                            workspace)
    if lens_out is None:
        lens_out = torch.empty_like(cache.lens)
    ws, ptr, n = _workspace(workspace, lambda: _evict_bytes(cache, keep, max_len), dev)
    st = lib().inf_kv_evict(cache.ref, pw,
                            pw if weights_out is None else _of(weights_out, "weights_out", torch.float32, dev, meta), pp,
                            pp if positions_out is None else _of(positions_out, "positions_out", torch.int32, dev, meta),
                            _of(lens_out, "lens_out", torch.int32, dev, (cache.rows,)), keep, int(recent), max_len, ptr,
                            n, _raw_stream(dev.index))
    _check(st, "inf_kv_evict")
    return lens_out


_select_sizes = {}


def _select_bytes(groups, beams, vocab):
    n = _select_sizes.get((groups, beams, vocab))
    if n is None:
        n = _select_sizes[groups, beams, vocab] = _size(lib().inf_beam_select_workspace, groups, beams, vocab)
    return n


def beam_select_workspace(groups, beams, vocab, device="cuda"):
    """A workspace for beam_select over these shapes."""
    return torch.empty(_select_bytes(groups, beams, vocab), dtype=torch.uint8, device=device)


def beam_select(logits, scores, finished=None, eos=None, workspace=None, stream=None):
    """(tokens, parents, scores, finished) of the best continuations: logits [groups * beams, vocab],
    scores float32 and finished int32 [groups, beams].  ``finished`` is None in the result
    where no ``eos`` is given."""
    dev = logits.device
    if scores.dim() != 2 or logits.dim() != 2 or logits.shape[0] != scores.numel():
        raise ValueError("beam_select: logits [groups * beams, vocab] and scores [groups, beams] expected")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"beam_select: float32 or bfloat16 logits expected, got {logits.dtype}")
    if finished is not None and eos is None:
        raise ValueError("beam_select: finished beams need eos")
    shape = scores.shape
    ps, pf = _of(scores, "scores", torch.float32, dev), _of(finished, "finished", torch.int32, dev, shape)
    if _elsewhere(dev, stream):
        with _on(dev, stream):
            return beam_select(logits, scores, finished, eos, workspace)
    vocab, (ld, step) = logits.shape[1], logits.stride()
    if vocab > 1 and step != 1:
        raise ValueError("beam_select: the logits of a row must be adjacent")
    groups, beams = shape
    tokens, parents = torch.empty_like(scores, dtype=torch.int32), torch.empty_like(scores, dtype=torch.int32)
    scores_out = torch.empty_like(scores)
    done = torch.empty_like(scores, dtype=torch.int32) if eos is not None else None
    ws, ptr, n = _workspace(workspace, lambda: _select_bytes(groups, beams, vocab), dev)
    st = lib().inf_beam_select(logits.data_ptr(), ld if logits.shape[0] > 1 else max(ld, vocab), ps, pf, groups, beams,
                               vocab, -1 if eos is None else int(eos), tokens.data_ptr(), parents.data_ptr(),
                               scores_out.data_ptr(), done.data_ptr() if done is not None else None, _dt(logits), ptr, n,
                               _raw_stream(dev.index))
    _check(st, "inf_beam_select")
    return tokens, parents, scores_out, done


def beam_reorder(cache, parents, spare, table_out=None, spare_out=None, stream=None):
    """(table, spare) after the rows of each group took over their parents' caches: parents int32
    [groups, beams], spare int32 [rows], one free page per row.  All layers of pools with a layer
    axis are done at once.  The cache's table is left; set ``cache.table`` to the new one."""
    dev = cache.device
    if parents.dim() != 2 or parents.numel() != cache.rows:
        raise ValueError("beam_reorder: parents [groups, beams] of the cache's rows expected")
    pp = _of(parents, "parents", torch.int32, dev)
    ps = _of(spare, "spare", torch.int32, dev, cache.lens.shape)
    if _elsewhere(dev, stream):
        with _on(dev, stream):
            return beam_reorder(cache, parents, spare, table_out, spare_out)
    shape = cache.table.shape
    if table_out is None:
        table_out = torch.empty_like(cache.table, memory_format=torch.contiguous_format)
        pt = table_out.data_ptr()
    else:
        pt = _of(table_out, "table_out", torch.int32, dev, shape)
    if spare_out is None:
        spare_out = torch.empty_like(spare)
        po = spare_out.data_ptr()
    else:
        po = _of(spare_out, "spare_out", torch.int32, dev, spare.shape)
    st = lib().inf_beam_reorder(cache.ref, cache.layers, *cache.layer_strides, pp, parents.shape[1],
                                pt, shape[1], ps, po, _raw_stream(dev.index))
    _check(st, "inf_beam_reorder")
    return table_out, spare_out


__all__ = ["PagedKV", "kv_append", "attn_decode_paged", "attn_decode_paged_workspace", "kv_evict",
           "kv_evict_workspace", "beam_select", "beam_select_workspace", "beam_reorder", "InfernoError"]
