"""Paged-cache operators on torch tensors (wraps include/lrrt_ops.h, which
describes them in full).

A cache is a pair of tensors per layer, keys and values of shape [pages,
page_size, kv_heads, head_dim], and a table of page numbers, one row per
sequence. Pages may be stored head by head: then pass the transposed view.

    ops = Ops()                                   # on the current stream
    q = ops.rope_append(q, k, v, keys[layer], values[layer], table, sequences,
                        positions, cos, sin)
    out, lse = ops.paged_attention(q, keys[layer], values[layer], table, lengths)
    scores, parents, tokens, finished = ops.beam_select(logits, scores, beams)
    table, lengths, status = ops.fork_pages(keys, values, table, lengths,
                                            parents.flatten())

Calls are enqueued on the stream that was current when the Ops was made, and
refuse to run while another is. Arguments that do not fit raise ValueError
before anything is enqueued, what the library refuses raises LrrtError.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import numpy as np
import torch

from . import native as N
from .qwen import Runtime

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# The argument structs of include/lrrt_ops.h, packed in one go (filling
# ctypes structures field by field costs more than a small launch);
# native.py declares them one by one.
_ROWS, _CACHE, _TABLE, _POOL = "Pqq", "PP6q5I4x", "Pq2I", "PP2q6I"
_ROPE = struct.Struct("@" + 4 * _ROWS + _CACHE + _TABLE + "4P6I")
_ATTENTION = struct.Struct("@" + 2 * _ROWS + _CACHE + _TABLE + "3P2I2f")
_FORK = struct.Struct("@" + _POOL + _TABLE + "4Pq2P2I")
_COMPACT = struct.Struct("@" + _POOL + _TABLE + "2PqP")
_COPY = struct.Struct("@" + _POOL + "2P2I")
_BEAM = struct.Struct("@Pq6P5Ii")
for _packed, _declared in ((_ROPE, N.RopeAppend), (_ATTENTION, N.PagedAttention),
                           (_FORK, N.PagesFork), (_COMPACT, N.PagesCompact),
                           (_COPY, N.PagesCopy), (_BEAM, N.BeamSelect)):
    assert _packed.size == C.sizeof(_declared)


def rope_tables(positions: int, rotary_dim: int, theta: float = 1.0e6, factor: float = 1.0,
                low_turns: float = 0.0, high_turns: float = 0.0, trained_positions: float = 0.0):
    """(cos, sin) of shape [positions, rotary_dim / 2] on the host, optionally
    scaled for contexts longer than the model was trained on (lro_rope_tables)."""
    cos = np.zeros((positions, rotary_dim // 2), np.float32)
    sin = np.zeros_like(cos)
    pointer = C.POINTER(C.c_float)
    N.check(N.operators().lro_rope_tables(positions, rotary_dim, theta, factor, low_turns,
                                          high_turns, trained_positions,
                                          cos.ctypes.data_as(pointer),
                                          sin.ctypes.data_as(pointer)), "lro_rope_tables")
    return cos, sin


def _refuse(text: str):
    raise ValueError(text)


class Ops:
    """The operators on one device and stream, with the workspace they share."""

    def __init__(self, device_index: int = 0):
        self.handle = self.queue = None
        device = Runtime.open_device(device_index)
        self.device = torch.device("cuda", device_index)
        self.stream = torch.cuda.current_stream(self.device)
        queue, handle = C.c_void_p(), C.c_void_p()
        N.check(N.runtime().lr_queue_wrap_stream(device, self.stream.cuda_stream,
                                                 C.byref(queue)), "lr_queue_wrap_stream")
        self.queue = queue
        image = N.OPS_CUBIN.read_bytes()
        N.check(N.operators().lro_context_create(device, queue, image, len(image),
                                                 C.byref(handle)), "lro_context_create")
        self.handle = handle
        self._index, self._raw_stream = device_index, self.stream.cuda_stream
        self._functions = {}
        for name in ("lro_rope_append", "lro_paged_attention", "lro_pages_fork",
                     "lro_pages_compact", "lro_pages_copy", "lro_beam_select"):
            # Their own prototypes: the arguments come as packed bytes.
            function = C.CFUNCTYPE(C.c_uint32, C.c_void_p, C.c_char_p)((name, N.operators()))
            self._functions[name] = function

    def close(self) -> None:
        if self.handle:
            N.check(N.operators().lro_context_destroy(self.handle), "lro_context_destroy")
            self.handle = None
        if self.queue:
            N.check(N.runtime().lr_queue_destroy(self.queue), "lr_queue_destroy")
            self.queue = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def reserve(self, workspace_bytes: int) -> None:
        """Workspace for later calls, so that none of them has to grow it."""
        N.check(N.operators().lro_context_reserve(self.handle, workspace_bytes),
                "lro_context_reserve")

    # ---- arguments -----------------------------------------------------------
    def _call(self, name: str, arguments: bytes) -> None:
        if not self.handle:
            _refuse("these operators are closed")
        if torch._C._cuda_getCurrentRawStream(self._index) != self._raw_stream:
            _refuse("the current stream is not the stream of these operators")
        status = self._functions[name](self.handle, arguments)
        if status != N.LR_SUCCESS:
            N.check(status, name)

    def _strides(self, t, name: str, dims: int, dtype):
        """The strides of a tensor on this device with contiguous last dimension."""
        strides = t.stride()
        if t.dtype is not dtype or t.get_device() != self._index or len(strides) != dims or \
                (strides[-1] != 1 and t.shape[-1] > 1):
            if t.device != self.device:
                _refuse(f"{name} is on {t.device}, not on {self.device}")
            if t.dtype != dtype:
                _refuse(f"{name} is {t.dtype}, not {dtype}")
            if t.dim() != dims:
                _refuse(f"{name} has {t.dim()} dimensions, not {dims}")
            _refuse(f"{name} is not contiguous in its last dimension")
        return strides

    def _vector(self, t, name: str, count: int, dtype) -> int:
        self._strides(t, name, 1, dtype)
        if t.numel() != count:
            _refuse(f"{name} has {t.numel()} elements, not {count}")
        return t.data_ptr()

    def _rows(self, t, name: str, shape, dtype):
        strides = self._strides(t, name, 3, dtype)
        if t.shape != shape:
            _refuse(f"{name} has the shape {tuple(t.shape)}, not {shape}")
        return t.data_ptr(), strides[0], strides[1]

    def _cache(self, keys, values):
        """(packed fields, type, shape) of one layer's pages."""
        dtype = keys.dtype
        if dtype not in _TYPES:
            _refuse(f"a cache of {dtype}")
        k = self._strides(keys, "keys", 4, dtype)
        v = self._strides(values, "values", 4, dtype)
        shape = keys.shape
        if shape != values.shape:
            _refuse("keys and values differ in shape")
        return (keys.data_ptr(), values.data_ptr(), k[0], k[1], k[2], v[0], v[1], v[2],
                _TYPES[dtype], *shape), dtype, shape

    def _table(self, table):
        strides = self._strides(table, "table", 2, torch.int32)
        return table.data_ptr(), strides[0], *table.shape

    def _pool(self, keys, values):
        """All layers' pages, [layers, pages, page_size, kv_heads, head_dim],
        each page contiguous, token by token or head by head."""
        if keys.dtype not in _TYPES:
            _refuse(f"a cache of {keys.dtype}")
        strides = self._strides(keys, "keys", 5, keys.dtype)
        if keys.shape != values.shape or self._strides(values, "values", 5, keys.dtype) != strides:
            _refuse("keys and values differ in shape or strides")
        layers, pages, size, heads, dim = keys.shape
        bytes_ = keys.element_size()
        layer, page, token, head, _ = strides
        if (token == heads * dim or size == 1) and (head == dim or heads == 1):
            segments, row = 1, heads * dim
        elif (token == dim or size == 1) and head == size * dim:
            segments, row = heads, dim
        else:
            return _refuse("pages must be contiguous, token by token or head by head")
        return (keys.data_ptr(), values.data_ptr(), layer * bytes_, page * bytes_, layers, pages,
                size, segments, row * bytes_, 0)

    # ---- operators -----------------------------------------------------------
    def rope_append(self, q, k, v, keys, values, table, sequences, positions, cos, sin,
                    interleaved: bool = False, out=None):
        """Rotates the queries [tokens, heads, head_dim] and keys [tokens,
        kv_heads, head_dim] by their positions and appends keys and values to
        the pages of their sequences (lro_rope_append). cos and sin: [positions,
        rotary_dim / 2], or None where nothing is rotated; sequences may be None:
        token t is of sequence t. Returns the queries, in `out` (may be q)."""
        cache, dtype, (_, _, kv_heads, dim) = self._cache(keys, values)
        q_rows = self._strides(q, "q", 3, dtype)
        tokens, heads, width = q.shape
        if width != dim:
            _refuse(f"q has a head_dim of {width}, the cache of {dim}")
        if out is None:
            out = q.new_empty((tokens, heads, dim))
            out_rows = (out.data_ptr(), heads * dim, dim)
        else:
            out_rows = self._rows(out, "out", (tokens, heads, dim), dtype)
        kv_shape = (tokens, kv_heads, dim)
        rotary = table_positions = cos_at = sin_at = 0
        if cos is not None:
            shape = cos.shape
            if self._strides(cos, "cos", 2, torch.float32) != \
                    self._strides(sin, "sin", 2, torch.float32) or shape != sin.shape or \
                    not cos.is_contiguous():
                _refuse("cos and sin must be contiguous and of one shape")
            table_positions, rotary = shape[0], 2 * shape[1]
            cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
        self._call("lro_rope_append", _ROPE.pack(
            q.data_ptr(), q_rows[0], q_rows[1], *out_rows, *self._rows(k, "k", kv_shape, dtype),
            *self._rows(v, "v", kv_shape, dtype), *cache, *self._table(table),
            0 if sequences is None else self._vector(sequences, "sequences", tokens, torch.int32),
            self._vector(positions, "positions", tokens, torch.int32), cos_at, sin_at, tokens,
            heads, rotary, table_positions, interleaved, 0))
        return out

    def paged_attention(self, q, keys, values, table, lengths, scale: Optional[float] = None,
                        softcap: float = 0.0, slopes=None, window: int = 0, out=None):
        """Attention of one query row per sequence, [rows, heads, head_dim], over
        the first lengths[row] tokens of its pages (lro_paged_attention). scale is
        head_dim ** -0.5 unless given; softcap, window: 0 for none; slopes:
        [heads] of a bias by distance, or None. Returns (out, lse)."""
        cache, dtype, (_, _, _, dim) = self._cache(keys, values)
        q_rows = self._strides(q, "q", 3, dtype)
        rows, heads, width = q.shape
        if width != dim:
            _refuse(f"q has a head_dim of {width}, the cache of {dim}")
        if out is None:
            out = q.new_empty((rows, heads, dim))
            out_rows = (out.data_ptr(), heads * dim, dim)
        else:
            out_rows = self._rows(out, "out", (rows, heads, dim), dtype)
        lse = q.new_empty((rows, heads), dtype=torch.float32)
        pages = self._table(table)
        if pages[2] != rows:
            _refuse(f"the table has {pages[2]} rows, not {rows}")
        if not 0 <= window < 2 ** 32:
            _refuse("window must be 0 or more, below 2^32")
        self._call("lro_paged_attention", _ATTENTION.pack(
            q.data_ptr(), q_rows[0], q_rows[1], *out_rows, *cache, *pages,
            self._vector(lengths, "lengths", rows, torch.int32),
            0 if slopes is None else self._vector(slopes, "slopes", heads, torch.float32),
            lse.data_ptr(), heads, window, dim ** -0.5 if scale is None else scale, softcap))
        return out, lse

    def fork_pages(self, keys, values, table, lengths, parents, room: int = 1, held=None,
                   table_out=None):
        """New sequences that continue their parents, copy-on-write, with pages
        for `room` more tokens (lro_pages_fork). keys and values are all layers'.
        Returns (table, lengths, status): status[0] pages were missing, status[1]
        are left free."""
        pool = self._pool(keys, values)
        pages = self._table(table)
        columns, count = pages[3], parents.numel()
        if table_out is None:
            table_out = table.new_empty((count, columns))
            out_stride = columns
        else:
            out_stride = self._strides(table_out, "table_out", 2, torch.int32)[0]
            if table_out.shape != (count, columns):
                _refuse(f"table_out has the shape {tuple(table_out.shape)}, not {(count, columns)}")
        if not 0 <= room < 2 ** 31:
            _refuse("room must be 0 or more, below 2^31")
        lengths_out = table.new_empty(count)
        status = table.new_empty(2)
        self._call("lro_pages_fork", _FORK.pack(
            *pool, *pages, self._vector(lengths, "lengths", pages[2], torch.int32),
            self._vector(parents, "parents", count, torch.int32),
            0 if held is None else self._vector(held, "held", pool[5], torch.uint8),
            table_out.data_ptr(), out_stride, lengths_out.data_ptr(), status.data_ptr(), count,
            room))
        return table_out, lengths_out, status

    def compact_pages(self, keys, values, table, held=None, table_out=None):
        """Live pages moved to the front of the pool (lro_pages_compact); table_out
        may be the table. Returns (table, status): status[0] pages are in use,
        status[1] were moved."""
        pool = self._pool(keys, values)
        pages = self._table(table)
        if table_out is None:
            table_out = table.new_empty(pages[2:])
        elif table_out.shape != table.shape:
            _refuse("table_out differs from the table in shape")
        status = table.new_empty(2)
        self._call("lro_pages_compact", _COMPACT.pack(
            *pool, *pages,
            0 if held is None else self._vector(held, "held", pool[5], torch.uint8),
            table_out.data_ptr(), self._strides(table_out, "table_out", 2, torch.int32)[0],
            status.data_ptr()))
        return table_out, status

    def copy_pages(self, keys, values, sources, targets) -> None:
        """Page sources[i] copied to page targets[i] in all layers (lro_pages_copy)."""
        pool = self._pool(keys, values)
        count = sources.numel()
        self._call("lro_pages_copy", _COPY.pack(
            *pool, self._vector(sources, "sources", count, torch.int32),
            self._vector(targets, "targets", count, torch.int32), count, 0))

    def beam_select(self, logits, scores, count: int, finished=None, end_token: int = -1):
        """The `count` best continuations of each group of beams from logits
        [groups, beams, vocab] and scores [groups, beams] (lro_beam_select).
        Returns (scores, parents, tokens, finished), each [groups, count];
        parents number the beams of all groups, as fork_pages takes them."""
        dtype = logits.dtype
        if dtype not in _TYPES:
            _refuse(f"logits of {dtype}")
        strides = self._strides(logits, "logits", 3, dtype)
        groups, beams, vocab = logits.shape
        if groups > 1 and beams > 1 and strides[0] != beams * strides[1]:
            _refuse("the rows of logits must be evenly spaced")
        for t, name, kind in ((scores, "scores", torch.float32),
                              (finished, "finished", torch.uint8)):
            if t is None and name == "finished":
                continue
            self._strides(t, name, 2, kind)
            if t.shape != (groups, beams) or not t.is_contiguous():
                _refuse(f"{name} must be contiguous, of shape {(groups, beams)}")
        if not 0 <= count < 2 ** 31:
            _refuse("count out of range")
        shape = (groups, count)
        scores_out = scores.new_empty(shape)
        parents = scores.new_empty(shape, dtype=torch.int32)
        tokens = scores.new_empty(shape, dtype=torch.int32)
        finished_out = scores.new_empty(shape, dtype=torch.uint8)
        self._call("lro_beam_select", _BEAM.pack(
            logits.data_ptr(), strides[1] if beams > 1 else strides[0], scores.data_ptr(),
            0 if finished is None else finished.data_ptr(), scores_out.data_ptr(),
            parents.data_ptr(), tokens.data_ptr(), finished_out.data_ptr(), _TYPES[dtype], groups,
            beams, vocab, count, end_token))
        return scores_out, parents, tokens, finished_out
