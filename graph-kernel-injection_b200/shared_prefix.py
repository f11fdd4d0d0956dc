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
import math
from typing import Optional, Tuple

import torch

import sbfa_native as native
import sparse_triton_kernel as stk

# how a row's attention to its own tokens comes to the merge (sbfa_prefix_attend)
OWN_NONE, OWN_16, OWN_32 = 0, 1, 2

_PROMPT_BLOCK = 128   # block size of the causal window mask behind attend_prompt


def no_gradients(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("this serving operator has no gradients: call it under torch.no_grad() "
                           "or with detached tensors")


def vector_readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` when its rows can be read in place in 16-byte pieces, else a contiguous copy."""
    st = t.stride()
    if st[-1] != 1 or t.data_ptr() % 16 or any(x < 0 or x % 8 for x in st[:-1]):
        return t.clone(memory_format=torch.contiguous_format)
    return t


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

    def _check(self, q: torch.Tensor) -> None:
        if (q.dim() != 4 or 0 in q.shape or q.shape[1] % self.heads
                or q.shape[3] != self.head_dim):
            raise ValueError(f"q must be [B, H, N, {self.head_dim}] with H a multiple of "
                             f"{self.heads}, got {tuple(q.shape)}")
        if q.device != self.device or q.dtype != self.dtype:
            raise ValueError(f"q must be {self.dtype} on {self.device}")
        no_gradients(q)

    def join(self, q: torch.Tensor, scale: float, own_o: Optional[torch.Tensor],
             own_lse: Optional[torch.Tensor], own_kind: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Attention of ``q`` ([B, H, N, D]) to the prefix, merged with its attention to its
        sequence's own tokens (``own_o``, ``own_lse`` in the form ``own_kind``, see
        ``sbfa_prefix_attend``): O and the natural-log LSE over both."""
        self._check(q)
        q = vector_readable(q)
        B, H, N, D = q.shape
        L = native.lib()
        dev = self.device
        o = torch.empty((B, H, N, D), dtype=self.dtype, device=dev)
        lse = torch.empty((B, H, N), dtype=torch.float32, device=dev)
        with native.device_guard(dev):
            need = int(L.sbfa_prefix_workspace_bytes(B, H, self.heads, N, self.length, D))
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
            native.check(L.sbfa_prefix_attend(
                q.data_ptr(), (ctypes.c_int64 * 3)(*q.stride()[:3]), self.k.data_ptr(),
                self.v.data_ptr(), native.ptr(own_o), native.ptr(own_lse), own_kind,
                o.data_ptr(), lse.data_ptr(), B, H, self.heads, N, self.length, D,
                native.dtype_code(self.dtype), scale, ws.data_ptr(), ws.numel(),
                native.stream_ptr(dev)), "prefix_attend")
        return o, lse

    def attend(self, q: torch.Tensor, softmax_scale: Optional[float] = None,
               return_lse: bool = False):
        """Attention of every query ([B, H, N, D]) to the whole prefix and nothing else:
        O ([B, H, N, D]) and, with ``return_lse``, the natural-log LSE ([B, H, N] fp32)."""
        scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
        o, lse = self.join(q, scale, None, None, OWN_NONE)
        return (o, lse) if return_lse else o

    def attend_prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window_size: int,
                      softmax_scale: Optional[float] = None, return_lse: bool = False):
        """Attention of the batch's own prompts behind the prefix: query ``i`` of a sequence
        ([B, H, N, D]) sees the whole prefix and the sequence's tokens ``(i - window_size, i]``
        of ``k``, ``v`` ([B, H_kv, N, D]).  Right-padded prompts need no lengths: no query
        sees a token behind it.  The own part runs the block-sparse forward, whose 16-bit O is
        merged with the prefix's."""
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
        no_gradients(k, v)
        scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
        if not 0 < scale <= 1e30:
            raise ValueError("softmax_scale must be positive and finite")
        tcore = stk._uses_tensor_cores(self.dtype, D)
        q, k, v = (stk._readable(t, tcore) for t in (q, k, v))
        o = torch.empty((B, H, N, D), dtype=self.dtype, device=self.device)
        lse = torch.empty((B, H, N), dtype=torch.float32, device=self.device)
        with native.device_guard(self.device):
            bm = _PROMPT_BLOCK
            mask = stk.make_streaming_mask(N, N, stk.StreamingMaskSpec(0, window_size), bm, bm,
                                           self.device)
            tm, tn = native.plan_tiles(0, self.dtype, D, N)
            plan = stk.build_plan(mask, N, N, bm, bm, tm, tn)
            native.check(native.lib().sbfa_fwd(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), B, H, N,
                N, D, native.dtype_code(self.dtype), scale, 1, 0, window_size, mask.data_ptr(),
                bm, bm, plan["row_ptr"].data_ptr(), plan["col_idx"].data_ptr(),
                stk._stride_array(q, k, v, o), self.heads, native.stream_ptr(self.device)), "fwd")
        o, lse = self.join(q, scale, o, lse, OWN_16)
        return (o, lse) if return_lse else o


__all__ = ["SharedPrefix"]
