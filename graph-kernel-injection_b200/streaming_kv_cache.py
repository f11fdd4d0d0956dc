"""StreamingLLM ring-buffer KV caches for the decode step: :class:`StreamingKVCache`
(16 or 32 bits, one length for the whole batch) and :class:`QuantizedStreamingKVCache`
(8 bits, ragged batches, grouped key/value heads).

No upstream counterpart: upstream decodes through its prefill kernel with
``N_Q = 1`` over the whole cache (``benchmark.py:799-804``), although the
StreamingLLM rule lets the query at position ``p`` see only positions
``[0, sink)`` and ``(p - window, p]``.  This cache keeps exactly those
``sink + window`` rows per (batch, head): row ``r < sink`` holds position
``r``; position ``p >= sink`` lives in row ``sink + (p - sink) % window``.
Decoding over it gives the same attention as the block-sparse decode over a
full-length cache (``block_sparse_attention`` with ``N_Q == 1``, causal,
``block_m = 1``), with ``(sink + window) / n_kv`` of the memory.

Either cache's ``attend`` takes a :class:`shared_prefix.SharedPrefix`, tokens that
every sequence of the batch has before its own and that are held once.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

import sbfa_native as native
from shared_prefix import (SharedPrefix, in_dual_level, no_gradients, stride_array,
                           vector_readable)


class StreamingKVCache:
    """Per-layer K/V ring cache, ``[B, H, sink + window, D]`` each, on one
    CUDA device.  ``append`` adds tokens in order; ``attend`` decodes the
    query of the last appended position."""

    def __init__(self, batch: int, heads: int, head_dim: int, sink_size: int, window_size: int,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda") -> None:
        if min(batch, heads, head_dim) <= 0:
            raise ValueError("batch, heads and head_dim must be positive")
        if sink_size < 0 or window_size < 0 or sink_size + window_size <= 0:
            raise ValueError("sink_size and window_size must be non-negative, not both zero")
        native.dtype_code(dtype)
        self.batch, self.heads, self.head_dim = batch, heads, head_dim
        self.sink_size, self.window_size = sink_size, window_size
        self.dtype = dtype
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        rows = sink_size + window_size
        self.k = torch.zeros(batch, heads, rows, head_dim, dtype=dtype, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.length = 0
        ws = int(native.lib().sbfa_ring_decode_workspace_bytes(batch, heads, head_dim, sink_size,
                                                               window_size))
        self._ws = torch.empty(max(ws, 16), dtype=torch.uint8, device=self.device)

    @property
    def memory_bytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    def _check(self, t: torch.Tensor, n: Optional[int], name: str) -> torch.Tensor:
        want = (self.batch, self.heads) + ((n,) if n is not None else (t.shape[2],)) + (
            self.head_dim,)
        if t.dim() != 4 or tuple(t.shape) != want:
            raise ValueError(f"{name} must have shape {want}, got {tuple(t.shape)}")
        if t.device != self.device or t.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}")
        return t.contiguous()

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Append K/V of the next ``k_new.shape[2]`` positions ([B, H, t, D])."""
        k_new = self._check(k_new, None, "k_new")
        v_new = self._check(v_new, k_new.shape[2], "v_new")
        n = k_new.shape[2]
        with torch.cuda.device(self.device):
            native.check(native.lib().sbfa_ring_append(
                self.k.data_ptr(), self.v.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
                self.batch, self.heads, self.head_dim, native.dtype_code(self.dtype),
                self.sink_size, self.window_size, self.length, n,
                native.stream_ptr(self.device)), "ring_append")
        self.length += n

    def attend(self, q: torch.Tensor, softmax_scale: Optional[float] = None,
               return_lse: bool = False, prefix: Optional[SharedPrefix] = None):
        """Attention of the query at position ``length - 1`` ([B, H, 1, D])
        over the cached sink and window; returns O ([B, H, 1, D]) and, with
        ``return_lse``, the natural-log LSE ([B, H, 1] fp32).  With ``prefix``
        the query sees that shared prefix as well (float16 / bfloat16)."""
        if self.length == 0:
            raise RuntimeError("the cache is empty: append the query's own token first")
        q = self._check(q, 1, "q")
        scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
        o = torch.empty_like(q)
        lse = torch.empty(self.batch, self.heads, 1, dtype=torch.float32, device=self.device)
        with torch.cuda.device(self.device):
            native.check(native.lib().sbfa_ring_decode(
                q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                self.batch, self.heads, self.head_dim, native.dtype_code(self.dtype), scale,
                self.sink_size, self.window_size, self.length, self._ws.data_ptr(),
                self._ws.numel(), native.stream_ptr(self.device)), "ring_decode")
        if prefix is not None:
            # o is rounded to its 16 bits before the merge rounds once more
            o, lse = prefix.join(q, scale, o, lse, return_lse)
        return (o, lse) if return_lse else o


_FORMATS = {"e4m3": (native.Q_E4M3, torch.float8_e4m3fn), "int8": (native.Q_INT8, torch.int8)}


class QuantizedStreamingKVCache:
    """Per-layer 8-bit K/V ring cache of ``sink_size + window_size`` rows per
    (sequence, head) on one CUDA device.

    Rows are quantised as they are appended: 8-bit codes (``fmt`` ``"e4m3"`` or
    ``"int8"``) and one power-of-two scale per row, the smallest that holds the
    row's largest magnitude, so the scaling itself is exact.  Every sequence has its
    own length, kept on the device in ``lengths`` (int64 [B]): batches may be
    ragged, and ``append`` / ``attend`` can be captured in a CUDA graph whose
    replays advance.  ``heads`` counts key/value heads; queries may have any
    multiple of it.  ``dtype`` (float16 or bfloat16) is the type of new rows, queries
    and outputs; ``head_dim`` is a multiple of 8, at most 256.

    ``k``, ``v`` (codes [B, H, rows, D]), ``scales`` (uint8 [B, H, rows, 2]: ``e + 127``
    of K's and of V's ``2 ** e``; 255 marks a row with a NaN or an infinity, which
    reads as NaN) and ``lengths`` are the state: save them, and hand them to :meth:`load`.
    No gradients.  Calls that write a cache (``append``, ``load``, ``reset``) and those around them
    follow each other on one stream; ``attend`` and ``read`` may overlap with each other.
    """

    def __init__(self, batch: int, heads: int, head_dim: int, sink_size: int, window_size: int,
                 dtype: torch.dtype = torch.bfloat16, fmt: str = "e4m3",
                 device: str | torch.device = "cuda") -> None:
        if min(batch, heads, head_dim) <= 0:
            raise ValueError("batch, heads and head_dim must be positive")
        if sink_size < 0 or window_size < 0 or sink_size + window_size <= 0:
            raise ValueError("sink_size and window_size must be non-negative, not both zero")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        if fmt not in _FORMATS:
            raise ValueError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
        row_bytes = int(native.lib().sbfa_qcache_row_bytes(head_dim))
        if row_bytes == 0:
            raise ValueError(f"head_dim must be a multiple of 8 and at most 256, got {head_dim}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("the cache must live on a CUDA device")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.batch, self.heads, self.head_dim = batch, heads, head_dim
        self.sink_size, self.window_size = sink_size, window_size
        self.dtype, self.fmt, self.device = dtype, fmt, dev
        rows = sink_size + window_size
        code, code_dtype = _FORMATS[fmt]
        self._k = torch.zeros(batch, heads, rows, row_bytes, dtype=torch.uint8, device=dev)
        self._v = torch.zeros_like(self._k)
        self._state = (self._k[..., :head_dim].view(code_dtype),
                       self._v[..., :head_dim].view(code_dtype),
                       torch.zeros(batch, heads, rows, 2, dtype=torch.uint8, device=dev),
                       torch.zeros(batch, dtype=torch.int64, device=dev))
        self._tickets = torch.zeros(batch, dtype=torch.int32, device=dev)
        self._scratch = {}   # scratch bytes of attend by the number of query heads
        self._struct = native.QCache(
            self._k.data_ptr(), self._v.data_ptr(), self.scales.data_ptr(),
            self.lengths.data_ptr(), self._tickets.data_ptr(), batch, heads, head_dim, sink_size,
            window_size, native.dtype_code(dtype), code)
        self._handle = ctypes.addressof(self._struct)

    # the tensors themselves, whose addresses the kernels hold: written to, never replaced
    @property
    def k(self) -> torch.Tensor:
        return self._state[0]

    @property
    def v(self) -> torch.Tensor:
        return self._state[1]

    @property
    def scales(self) -> torch.Tensor:
        return self._state[2]

    @property
    def lengths(self) -> torch.Tensor:
        return self._state[3]

    @property
    def memory_bytes(self) -> int:
        return 2 * self._k.numel() + self.scales.numel()

    def _check(self, t: torch.Tensor, shape: Tuple[int, ...], name: str) -> None:
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}")
        if t.requires_grad or in_dual_level():
            no_gradients(t)

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
        """Quantise and append the next ``t`` tokens of every sequence ([B, H, t, D],
        views welcome).  ``counts`` (int64, or int32, [B] on the device, clamped to [0, t]) says how many
        of them each sequence takes: the rest of a right-padded batch is not read."""
        shape = k_new.shape
        if len(shape) != 4:
            raise ValueError(f"k_new must be [B, H, t, D], got {tuple(shape)}")
        n = shape[2]
        shape = (self.batch, self.heads, n, self.head_dim)
        self._check(k_new, shape, "k_new")
        self._check(v_new, shape, "v_new")
        if counts is not None:
            if (tuple(counts.shape) != (self.batch,) or counts.device != self.device
                    or counts.dtype not in (torch.int64, torch.int32)):
                raise ValueError(f"counts must be int64 or int32 [{self.batch}] on {self.device}")
            counts = counts.to(torch.int64).contiguous()
        if n == 0:
            return
        k_new, v_new = vector_readable(k_new), vector_readable(v_new)
        strides = stride_array(k_new.stride()[:3] + v_new.stride()[:3])
        native.launch("sbfa_qcache_append", self.device, self._handle, k_new.data_ptr(),
                      v_new.data_ptr(), strides, None if counts is None else counts.data_ptr(), n)

    def attend(self, q: torch.Tensor, softmax_scale: Optional[float] = None,
               return_lse: bool = False, prefix: Optional[SharedPrefix] = None):
        """Attention of each sequence's query at its last position ([B, Hq, 1, D], Hq a
        multiple of ``heads``) over its cached rows; returns O ([B, Hq, 1, D]) and, with
        ``return_lse``, the natural-log LSE ([B, Hq, 1] fp32).  A sequence that has no
        token yet gives zeros.  With ``prefix`` every query sees that shared prefix as
        well: the merged result is rounded once."""
        shape = q.shape
        hq = shape[1] if len(shape) == 4 else 0
        if hq == 0 or hq % self.heads:
            raise ValueError(f"q must be [B, Hq, 1, D] with Hq a multiple of {self.heads}, got "
                             f"{tuple(shape)}")
        self._check(q, (self.batch, hq, 1, self.head_dim), "q")
        scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
        q = q.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        if prefix is not None:
            return prefix.attend_cached(self, q, scale, return_lse)
        need = self._scratch.get(hq)
        if need is None:
            with native.device_guard(self.device):
                need = self._scratch[hq] = native.lib().sbfa_qcache_attend_workspace_bytes(
                    self._handle, hq)
        o = torch.empty_like(q)
        lse = ws = None
        if return_lse:
            lse = torch.empty(self.batch, hq, 1, dtype=torch.float32, device=self.device)
        if need > 0:   # from torch's allocator, so of the call's stream or graph
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        native.launch("sbfa_qcache_attend", self.device, self._handle, q.data_ptr(), o.data_ptr(),
                      None if lse is None else lse.data_ptr(), hq, scale,
                      None if ws is None else ws.data_ptr(), need)
        return (o, lse) if return_lse else o

    def read(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The kept rows as ``dtype`` values in order of position: K and V
        ([B, H, rows, D], row i = the sequence's i-th kept position, zeros behind the
        last) and those positions (int64 [B, rows], -1 behind the last)."""
        rows = self.sink_size + self.window_size
        k = torch.empty(self.batch, self.heads, rows, self.head_dim, dtype=self.dtype,
                        device=self.device)
        v = torch.empty_like(k)
        positions = torch.empty(self.batch, rows, dtype=torch.int64, device=self.device)
        native.launch("sbfa_qcache_read", self.device, self._handle, k.data_ptr(), v.data_ptr(),
                      positions.data_ptr())
        return k, v, positions

    def load(self, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor,
             lengths: torch.Tensor) -> None:
        """Take over a saved state (the tensors ``k``, ``v``, ``scales``, ``lengths`` of a cache
        of the same geometry and format).  Waits for the device to check the lengths."""
        for t, mine, name in ((k, self.k, "k"), (v, self.v, "v"), (scales, self.scales, "scales"),
                              (lengths, self.lengths, "lengths")):
            if t.shape != mine.shape:
                raise ValueError(f"{name} must have shape {tuple(mine.shape)}, got "
                                 f"{tuple(t.shape)}")
            # codes may also come as the bytes they are
            if t.dtype != mine.dtype and not (name in ("k", "v") and t.dtype == torch.uint8):
                raise ValueError(f"{name} must hold {mine.dtype}, got {t.dtype}")
        if bool((lengths < 0).any()):
            raise ValueError("lengths must not be negative")
        self._k[..., :self.head_dim].copy_(k.view(torch.uint8))
        self._v[..., :self.head_dim].copy_(v.view(torch.uint8))
        self.scales.copy_(scales)
        self.lengths.copy_(lengths)

    def reset(self, sequences=None) -> None:
        """Forget every sequence, or those that ``sequences`` (indices or a bool mask) names."""
        if sequences is None:
            self.lengths.zero_()
        else:
            self.lengths[sequences] = 0
