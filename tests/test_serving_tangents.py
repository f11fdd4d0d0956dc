"""The serving operators have no gradients of either mode: a dual tensor is refused, not taken as its
primal."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from shared_prefix import SharedPrefix, no_gradients
from streaming_kv_cache import QuantizedStreamingKVCache, StreamingKVCache


def test_a_tangent_is_refused():
    x = torch.randn(2, 3)
    no_gradients(x)
    with forward_ad.dual_level():
        no_gradients(x, x)
        with pytest.raises(RuntimeError, match="forward-mode gradients"):
            no_gradients(x, forward_ad.make_dual(x, x))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode gradients"):
            no_gradients(forward_ad.make_dual(x, x))
    no_gradients(x)


@pytest.mark.gpu
def test_entry_points_refuse_a_tangent():
    dt, dev = torch.float16, "cuda"
    x = torch.randn(1, 2, 3, 64, dtype=dt, device=dev)
    q = x[:, :, :1].contiguous()
    pre = SharedPrefix(x[0], x[0])
    cache = QuantizedStreamingKVCache(1, 2, 64, 0, 8, dtype=dt, device=dev)
    ring = StreamingKVCache(1, 2, 64, 0, 8, dtype=dt, device=dev)
    cache.append(x, x)
    ring.append(x, x)
    with forward_ad.dual_level():
        d, dq = forward_ad.make_dual(x, x), forward_ad.make_dual(q, q)
        for call in (lambda: cache.append(d, x), lambda: cache.append(x, d),
                     lambda: cache.attend(dq), lambda: cache.attend(dq, prefix=pre),
                     lambda: ring.attend(dq, prefix=pre), lambda: pre.attend(d),
                     lambda: pre.attend_prompt(d, x, x, 2), lambda: pre.attend_prompt(x, d, x, 2),
                     lambda: pre.attend_prompt(x, x, d, 2), lambda: SharedPrefix(d[0], x[0])):
            with pytest.raises(RuntimeError, match="forward-mode gradients"):
                call()
        cache.append(x, x)
        assert torch.equal(cache.attend(q), cache.attend(forward_ad.unpack_dual(dq).primal))
    assert cache.lengths.tolist() == [6]
