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
refuse to run while another is. Threads may share an Ops: their calls are
enqueued one after another. There is no backward pass: tensors that require
gradients are refused where these are recorded. Arguments that do not fit raise ValueError
before anything is enqueued, what the library refuses raises LrrtError.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
from typing import Optional

import numpy as np
import torch

from . import native as N
from .qwen import Runtime


def _load_binding():
    N.operators()
    if not N.OPS_TORCH_PATH.exists():
        raise RuntimeError(f"{N.OPS_TORCH_PATH} is missing: run light-rocm-runtime_b200/build.py")
    spec = importlib.util.spec_from_file_location("lrrt_ops_torch", N.OPS_TORCH_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_binding = _load_binding()


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


class Ops:
    """The operators on one device and stream, with the workspace they share."""

    def __init__(self, device_index: int = 0):
        self.handle = self.queue = None
        self.device = torch.device("cuda", device_index)
        with torch.cuda.device(self.device):  # the library makes its device current
            self._open(device_index)

    def _open(self, device_index: int) -> None:
        device = Runtime.open_device(device_index)
        self.stream = torch.cuda.current_stream(self.device)
        queue, handle = C.c_void_p(), C.c_void_p()
        N.check(N.runtime().lr_queue_wrap_stream(device, self.stream.cuda_stream,
                                                 C.byref(queue)), "lr_queue_wrap_stream")
        self.queue = queue
        image = N.OPS_CUBIN.read_bytes()
        N.check(N.operators().lro_context_create(device, queue, image, len(image),
                                                 C.byref(handle)), "lro_context_create")
        self.handle = handle
        self._ops = _binding.open(handle.value, device_index, N.check)

    def close(self) -> None:
        with torch.cuda.device(self.device):
            self._close()

    def _close(self) -> None:
        if self.handle:
            _binding.close(self._ops)
            N.check(N.operators().lro_context_destroy(self.handle), "lro_context_destroy")
            self.handle = None
        if self.queue:
            N.check(N.runtime().lr_queue_destroy(self.queue), "lr_queue_destroy")
            self.queue = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def reserve(self, workspace_bytes: int, counters: int = 0) -> None:
        """Workspace and counters for later calls, so that none of them has to
        grow them, which a call that is captured cannot (lro_context_create
        says what calls need)."""
        _binding.reserve(self._ops, workspace_bytes, counters)

    # ---- operators -----------------------------------------------------------
    def rope_append(self, q, k, v, keys, values, table, sequences, positions, cos, sin,
                    interleaved: bool = False, out=None):
        """Rotates the queries [tokens, heads, head_dim] and keys [tokens,
        kv_heads, head_dim] by their positions and appends keys and values to
        the pages of their sequences (lro_rope_append). cos and sin: [positions,
        rotary_dim / 2], or None where nothing is rotated; sequences may be None:
        token t is of sequence t. Returns the queries, in `out` (may be q)."""
        return _binding.rope_append(self._ops, q, k, v, keys, values, table, sequences, positions,
                                    cos, sin, interleaved, out)

    def paged_attention(self, q, keys, values, table, lengths, scale: Optional[float] = None,
                        softcap: float = 0.0, slopes=None, window: int = 0, out=None):
        """Attention of one query row per sequence, [rows, heads, head_dim], over
        the first lengths[row] tokens of its pages (lro_paged_attention). scale is
        head_dim ** -0.5 unless given; softcap, window: 0 for none; slopes:
        [heads] of a bias by distance, or None. Returns (out, lse)."""
        return _binding.paged_attention(self._ops, q, keys, values, table, lengths, scale,
                                        softcap, slopes, window, out)

    def fork_pages(self, keys, values, table, lengths, parents, room: int = 1, held=None,
                   table_out=None):
        """New sequences that continue their parents, copy-on-write, with pages
        for `room` more tokens (lro_pages_fork). keys and values are all layers'.
        Returns (table, lengths, status): status[0] pages were missing, status[1]
        are left free."""
        return _binding.fork_pages(self._ops, keys, values, table, lengths, parents, room, held,
                                   table_out)

    def compact_pages(self, keys, values, table, held=None, table_out=None):
        """Live pages moved to the front of the pool (lro_pages_compact); table_out
        may be the table. Returns (table, status): status[0] pages are in use,
        status[1] were moved."""
        return _binding.compact_pages(self._ops, keys, values, table, held, table_out)

    def copy_pages(self, keys, values, sources, targets) -> None:
        """Page sources[i] copied to page targets[i] in all layers (lro_pages_copy)."""
        _binding.copy_pages(self._ops, keys, values, sources, targets)

    def beam_select(self, logits, scores, count: int, finished=None, end_token: int = -1):
        """The `count` best continuations of each group of beams from logits
        [groups, beams, vocab] and scores [groups, beams] (lro_beam_select).
        Returns (scores, parents, tokens, finished), each [groups, count];
        parents number the beams of all groups, as fork_pages takes them."""
        return _binding.beam_select(self._ops, logits, scores, count, finished, end_token)
