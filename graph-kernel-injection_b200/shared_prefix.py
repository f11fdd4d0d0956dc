"""Attention of a batch to a prefix that all its sequences share.

No upstream counterpart.  A system prompt, a document or a set of examples that
stands before every sequence of a batch is held once ([H_kv, P, D]) instead of
once per sequence, and its K and V are read once per call for the whole batch:
every query sees every prefix token, so the queries of all sequences and of a
key/value head's group make the rows of one tensor-core matrix product.  In
StreamingLLM terms the prefix is a set of sinks that the batch shares; the
sequence's own tokens follow it under the causal window rule.

* decode: ``StreamingKVCache.attend(q, prefix=...)`` or
  ``QuantizedStreamingKVCache.attend(q, prefix=...)``;
* prompts: :meth:`SharedPrefix.attend_prompt`;
* the prefix alone: :meth:`SharedPrefix.attend`.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad

import sbfa_native as native
import sparse_triton_kernel as stk


def no_gradients(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("this serving operator has no gradients: call it under torch.no_grad() "
                           "or with detached tensors")
    if in_dual_level() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("this serving operator has no forward-mode gradients: call it with the "
                           "primals")


def in_dual_level() -> bool:
    """Whether tensors may carry tangents at all."""
    return forward_ad._current_level >= 0


def vector_readable(t: torch.Tensor) -> torch.Tensor:
    """The 4-D ``t`` when its rows can be read in place in 16-byte pieces, else a contiguous copy."""
    b, h, n, d = t.stride()
    if d != 1 or (b | h | n) & 7 or t.data_ptr() & 15:
        return t.clone(memory_format=torch.contiguous_format)
    return t


@functools.lru_cache(maxsize=256)
def stride_array(strides: Tuple[int, ...]):
    """A host array of these element strides for the C ABI, which only reads it."""
    return (ctypes.c_int64 * len(strides))(*strides)


def tma_readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` when tiles of it can be fetched in place, else a contiguous copy."""
    t = stk._readable(t, True)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


class SharedPrefix:
    """K and V ([H_kv, P, D], float16 or bfloat16, D a multiple of 8 and at most 128) of
    the tokens that stand before every sequence of a batch.  Contiguous tensors are
    kept as they are (later writes to them are seen), others are copied.  No gradients."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor) -> None:
        if k.dim() != 3 or k.shape != v.shape or 0 in k.shape:
            raise ValueError("k and v must both be [H_kv, P, D] with no empty dimension")
        if not (k.is_cuda and k.device == v.device):
            raise ValueError("k and v must live on the same CUDA device")
        if k.dtype != v.dtype or k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("k and v must share dtype float16 or bfloat16")
        if k.shape[2] % 8 or k.shape[2] > 128:
            raise ValueError(f"head_dim must be a multiple of 8 and at most 128, got {k.shape[2]}")
        no_gradients(k, v)
        native.lib()
        self.k, self.v = (t if t.is_contiguous() and t.data_ptr() % 16 == 0
                          else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        self.heads, self.length, self.head_dim = (int(x) for x in k.shape)
        self.dtype, self.device = k.dtype, k.device
        self._code = native.dtype_code(k.dtype)
        self._scratch: Dict[tuple, int] = {}   # scratch bytes by a call's sizes

    def _check(self, q: torch.Tensor) -> None:
        if (q.dim() != 4 or 0 in q.shape or q.shape[1] % self.heads
                or q.shape[3] != self.head_dim):
            raise ValueError(f"q must be [B, H, N, {self.head_dim}] with H a multiple of "
                             f"{self.heads}, got {tuple(q.shape)}")
        if q.device != self.device or q.dtype != self.dtype:
            raise ValueError(f"q must be {self.dtype} on {self.device}")
        no_gradients(q)

    def join(self, q: torch.Tensor, scale: float, own_o: Optional[torch.Tensor],
             own_lse: Optional[torch.Tensor],
             return_lse: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """Attention of ``q`` ([B, H, N, D]) to the prefix, merged with its attention to its
        sequence's own tokens where ``own_o``, ``own_lse`` give it (every query saw a
        token there): O and, with ``return_lse``, the natural-log LSE over both."""
        self._check(q)
        q = vector_readable(q)
        B, H, N, D = q.shape
        dev = self.device
        o = torch.empty(B, H, N, D, dtype=self.dtype, device=dev)
        lse = torch.empty(B, H, N, dtype=torch.float32, device=dev) if return_lse else None
        ws, ws_bytes = self._workspace(B, H, N, 0)
        native.launch("sbfa_prefix_attend", dev, q.data_ptr(), stride_array(q.stride()[:3]),
                      self.k.data_ptr(), self.v.data_ptr(), native.ptr(own_o),
                      native.ptr(own_lse), o.data_ptr(), native.ptr(lse), B, H, self.heads, N,
                      self.length, D, self._code, scale, native.ptr(ws), ws_bytes)
        return o, lse

    def _workspace(self, B: int, H: int, N: int, window: int):
        """Scratch of one call (from torch's allocator, so of its stream or graph) and its bytes."""
        need = self._scratch.get((B, H, N, window))
        if need is None:
            with native.device_guard(self.device):
                need = self._remember((B, H, N, window), native.lib().sbfa_prefix_workspace_bytes(
                    B, H, self.heads, N, self.length, self.head_dim, window))
        if need <= 0:   # none, or a bad shape that the call refuses
            return None, 0
        return torch.empty(need, dtype=torch.uint8, device=self.device), need

    def _remember(self, sizes: tuple, need: int) -> int:
        if len(self._scratch) >= 256:
            self._scratch.clear()
        self._scratch[sizes] = need
        return need

    def attend_cached(self, cache, q: torch.Tensor, scale: float, return_lse: bool):
        """A decode step of a ``QuantizedStreamingKVCache`` behind this prefix (``q`` checked by the
        cache)."""
        if (cache.heads != self.heads or cache.head_dim != self.head_dim
                or cache.dtype != self.dtype or cache.device != self.device):
            raise ValueError(f"the prefix has {self.heads} heads of {self.head_dim} {self.dtype} on "
                             f"{self.device}, the cache {cache.heads} of {cache.head_dim} "
                             f"{cache.dtype} on {cache.device}")
        B, H = q.shape[:2]
        dev = self.device
        o = torch.empty_like(q)
        lse = torch.empty(B, H, 1, dtype=torch.float32, device=dev) if return_lse else None
        sizes = (B, H, cache.sink_size, cache.window_size, "cache")
        need = self._scratch.get(sizes)
        if need is None:
            with native.device_guard(dev):
                need = self._remember(sizes, native.lib().sbfa_qcache_prefix_workspace_bytes(
                    cache._handle, H, self.length))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        native.launch("sbfa_qcache_prefix_attend", dev, cache._handle, q.data_ptr(),
                      self.k.data_ptr(), self.v.data_ptr(), self.length, o.data_ptr(),
                      native.ptr(lse), H, scale, ws.data_ptr(), need)
        return (o, lse) if return_lse else o

    def attend(self, q: torch.Tensor, softmax_scale: Optional[float] = None,
               return_lse: bool = False):
        """Attention of every query ([B, H, N, D]) to the whole prefix and nothing else:
        O ([B, H, N, D]) and, with ``return_lse``, the natural-log LSE ([B, H, N] fp32)."""
        scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
        o, lse = self.join(q, scale, None, None, return_lse)
        return (o, lse) if return_lse else o

    def attend_prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window_size: int,
                      softmax_scale: Optional[float] = None, return_lse: bool = False,
                      sink_size: int = 0):
        """Attention of the batch's own prompts behind the prefix: query ``i`` of a sequence
        ([B, H, N, D]) sees the whole prefix and the sequence's tokens ``(i - window_size, i]``
        and, of the first ``sink_size``, those up to ``i``, of ``k``, ``v`` ([B, H_kv, N, D]; views
        welcome).  Give the two sizes of the cache that goes on from the prompt: behind a prefix it
        shows its sinks to every later token.  Right-padded prompts need no lengths: no query sees
        a token behind it.  One pass over both parts."""
        self._check(q)
        B, H, N, D = q.shape
        if tuple(k.shape) != (B, self.heads, N, D) or k.shape != v.shape:
            raise ValueError(f"k and v must have shape {(B, self.heads, N, D)}, got "
                             f"{tuple(k.shape)} and {tuple(v.shape)}")
        for t in (k, v):
            if t.device != self.device or t.dtype != self.dtype:
                raise ValueError(f"k and v must be {self.dtype} on {self.device}")
        if window_size < 1:
            raise ValueError("window_size must be at least 1: a query sees its own token")
        if sink_size < 0:
            raise ValueError("sink_size must not be negative")
        no_gradients(k, v)
        scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
        q, k, v = vector_readable(q), tma_readable(k), tma_readable(v)
        dev = self.device
        o = torch.empty(B, H, N, D, dtype=self.dtype, device=dev)
        lse = torch.empty(B, H, N, dtype=torch.float32, device=dev) if return_lse else None
        ws, ws_bytes = self._workspace(B, H, N, window_size)
        strides = stride_array((*q.stride()[:3], *stk._strides3(k), *stk._strides3(v)))
        native.launch("sbfa_prefix_prompt_sinks", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), strides,
                      self.k.data_ptr(), self.v.data_ptr(), o.data_ptr(), native.ptr(lse), B, H,
                      self.heads, N, self.length, D, self._code, scale, sink_size, window_size,
                      native.ptr(ws), ws_bytes)
        return (o, lse) if return_lse else o


__all__ = ["SharedPrefix"]
