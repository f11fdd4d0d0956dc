"""Prompts behind a shared prefix: infinities that meet slices of a row's keys, padding, and sinks,
against 64 bits within the bounds of ``serving_reference``."""

from __future__ import annotations

import math

import pytest
import torch

import sbfa_native as native
from streaming_kv_cache import QuantizedStreamingKVCache, StreamingKVCache
from tests import serving_reference as ref
from tests.test_gpu_quantized_cache import gen, rows
from tests.test_gpu_shared_prefix import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,G,N,P,D,W,at", [
    (1, 2, 600, 3333, 64, 50, (100, 520)),      # slices, the flagged ones far from the first keys
    (1, 1, 900, 9000, 128, 300, (10, 700)),
    (3, 1, 64, 5000, 128, 64, (5, 60)),
    (2, 2, 300, 100, 64, 40, (20, 250)),        # few keys
])
def test_an_infinity_stays_one_whatever_other_slices_hold(dtype, B, G, N, P, D, W, at):
    """Two value rows of one sequence hold non-finite elements: the queries that see one of them get
    it as it is, in its column, and every other output is what finite rows give."""
    g = gen(50)
    pre = make(g, 1, P, D, dtype)
    q, k, v = (rows(g, (B, N, h, D), dtype, 0.2).transpose(1, 2) for h in (G, 1, 1))
    clean = pre.attend_prompt(q, k, v, window_size=W)
    v = v.clone()
    first, second = at
    v[0, 0, first, 3], v[0, 0, first, 9] = math.inf, -math.inf
    v[0, 0, second, 3], v[0, 0, second, 7] = math.inf, math.nan
    o = pre.attend_prompt(q, k, v, window_size=W)
    want = clean.clone()
    want[0, :, first:first + W, 3] = math.inf
    want[0, :, first:first + W, 9] = -math.inf
    want[0, :, second:second + W, 3] = math.inf
    want[0, :, second:second + W, 7] = math.nan
    same = (o == want) | (torch.isnan(o) & torch.isnan(want))
    assert same.all(), f"{(~same).sum().item()} differ, first at {(~same).nonzero()[0].tolist()}"
    assert native.device_status() == 0


def expected(pre, q, k, v, b, h, G, W, S=0, n=None):
    """O, LSE, the weighted mean of |v| and the scores' error of head h of sequence b over its first n
    tokens."""
    N, D = (q.shape[2] if n is None else n), q.shape[3]
    i = torch.arange(N, device=DEV)
    gap = i[:, None] - i[None, :]
    own = (gap >= 0) & ((gap < W) | (i[None, :] < S))
    seen = torch.cat((torch.ones(N, pre.length, dtype=torch.bool, device=DEV), own), 1)
    kk = torch.cat((pre.k[h // G], k[b, h // G, :N])).double()
    vv = torch.cat((pre.v[h // G], v[b, h // G, :N])).double()
    qq = q[b, h, :N].double()
    x = (qq @ kk.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
    w = torch.softmax(x, -1)
    ds = (qq.abs() @ kk.abs().T).amax(-1) / math.sqrt(D) * D * 2.0 ** -23
    return w @ vv, torch.logsumexp(x, -1), w @ vv.abs(), ds


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,G,N,P,D,W,S", [
    (2, 2, 4, 100, 300, 128, 16, 4), (37, 1, 2, 5, 200, 64, 1, 2), (9, 1, 5, 64, 128, 40, 3, 1),
    (3, 1, 7, 65, 64, 96, 5, 30), (2, 2, 1, 513, 5, 128, 20, 1), (1, 1, 1, 700, 1500, 64, 16, 200),
    (1, 2, 1, 900, 1000, 128, 100, 129), (2, 1, 2, 600, 3333, 64, 7, 4),   # slices
    (3, 1, 1, 300, 50, 64, 40, 1000), (5, 1, 1, 129, 9000, 128, 2, 128), (150, 2, 1, 1, 10, 128, 7, 3),
    (1, 1, 1, 1500, 64, 128, 64, 1)])
def test_prompts_with_own_sinks(dtype, B, Hkv, G, N, P, D, W, S):
    g = gen(52)
    pre = make(g, Hkv, P, D, dtype)
    q, k, v = (rows(g, (B, N, h, D), dtype, 0.2).transpose(1, 2) for h in (Hkv * G, Hkv, Hkv))
    o, lse = pre.attend_prompt(q, k, v, window_size=W, sink_size=S, return_lse=True)
    u = ref.half_step(dtype)
    for b in range(B):
        for h in range(Hkv * G):
            eo, el, A, ds = expected(pre, q, k, v, b, h, G, W, S)
            ref.check(o[b, h], eo, A, ds, u, u, label=f"b{b} h{h}")
            ref.check_lse(lse[b, h], el, ds, f"b{b} h{h}")
    assert native.device_status() == 0


@pytest.mark.parametrize("B,G,N,P,W,S", [(1, 2, 600, 3333, 50, 3), (2, 1, 60, 100, 7, 2),
                                         (1, 1, 800, 40, 100, 140)])
def test_an_infinity_in_a_sink_reaches_every_later_query(B, G, N, P, W, S):
    g = gen(53)
    D, dtype = 64, torch.bfloat16
    pre = make(g, 1, P, D, dtype)
    q, k, v = (rows(g, (B, N, h, D), dtype, 0.2).transpose(1, 2) for h in (G, 1, 1))
    clean = pre.attend_prompt(q, k, v, window_size=W, sink_size=S)
    v = v.clone()
    at = N - N // 8                    # an ordinary token near the end
    v[0, 0, S - 1, 3], v[0, 0, at, 7] = math.inf, math.nan
    o = pre.attend_prompt(q, k, v, window_size=W, sink_size=S)
    want = clean.clone()
    want[0, :, S - 1:, 3] = math.inf
    want[0, :, at:at + W, 7] = math.nan
    same = (o == want) | (torch.isnan(o) & torch.isnan(want))
    assert same.all(), f"{(~same).sum().item()} differ, first at {(~same).nonzero()[0].tolist()}"


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16)])
@pytest.mark.parametrize("S,W", [(4, 30), (0, 50), (130, 20)])
def test_prefill_and_decode_behind_a_prefix_see_the_same(fmt, dtype, S, W):
    """A prompt's last query and the decode step of a cache that holds the same prompt: both
    within their bounds of one 64-bit result, for either cache, and the token after it."""
    g = gen(54)
    B, H, G, N, P, D = 2, 2, 3, 200, 300, 64
    pre = make(g, H, P, D, dtype)
    whole = QuantizedStreamingKVCache(B, H, D, 0, N + 1, dtype=dtype, fmt=fmt, device=DEV)
    whole.append(*(rows(g, (B, H, N + 1, D), dtype, 0.2) for _ in range(2)))
    k, v, _ = whole.read()             # values that 8 bits hold exactly
    q = rows(g, (B, H * G, N + 1, D), dtype, 0.2)
    o, lse = pre.attend_prompt(q, k, v, window_size=W, sink_size=S, return_lse=True)
    small = QuantizedStreamingKVCache(B, H, D, S, W, dtype=dtype, fmt=fmt, device=DEV)
    wide = StreamingKVCache(B, H * G, D, S, W, dtype=dtype, device=DEV)
    u = ref.half_step(dtype)
    start = 0
    for n in (N, N + 1):
        small.append(k[:, :, start:n], v[:, :, start:n])
        wide.append(*(x[:, :, start:n].repeat_interleave(G, 1) for x in (k, v)))
        start = n
        d8 = small.attend(q[:, :, n - 1:n], return_lse=True, prefix=pre)
        d16 = wide.attend(q[:, :, n - 1:n], return_lse=True, prefix=pre)
        for b in range(B):
            for h in range(H * G):
                eo, el, A, ds = (x[n - 1:n] for x in expected(pre, q, k, v, b, h, G, W, S))
                big = v[b, h // G].abs().max().item()
                ref.check(o[b, h, n - 1:n], eo, A, ds, u, u, label="prompt")
                ref.check(d8[0][b, h], eo, A, ds, u, max(u, ref.U16), n * 2.0 ** -25 * big, "8 bits")
                # the 16-bit ring's own part is rounded once before the merge: u A more
                ref.check(d16[0][b, h], eo, A, ds, u, 2 * u, label="16 bits")
                for got in (lse[b, h, n - 1:n], d8[1][b, h], d16[1][b, h]):
                    ref.check_lse(got, el, ds)


def test_sink_size_must_not_be_negative():
    pre = make(gen(55), 1, 10, 64, torch.float16)
    x = torch.zeros(1, 1, 3, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="sink_size"):
        pre.attend_prompt(x, x, x, window_size=2, sink_size=-1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,n,P,W", [(64, 17, 200, 40), (300, 129, 77, 50), (700, 1, 3000, 256)])
def test_padding_reaches_no_query_of_the_prompt(dtype, N, n, P, W):
    """A padded prompt and the prompt alone both hold the bound of the 64-bit result."""
    g = gen(51)
    B, Hkv, G, D = 3, 2, 4, 128
    u = ref.half_step(dtype)
    pre = make(g, Hkv, P, D, dtype)
    q, k, v = (rows(g, (B, h, N, D), dtype, 0.2) for h in (Hkv * G, Hkv, Hkv))
    padded = pre.attend_prompt(q, k, v, window_size=W, return_lse=True)
    alone = pre.attend_prompt(q[1:2, :, :n], k[1:2, :, :n], v[1:2, :, :n], window_size=W,
                              return_lse=True)
    for h in range(Hkv * G):
        eo, el, A, ds = expected(pre, q, k, v, 1, h, G, W, n=n)
        for (o, lse), b in ((padded, 1), (alone, 0)):
            ref.check(o[b, h, :n], eo, A, ds, u, u, label=f"h{h} b{b}")
            ref.check_lse(lse[b, h, :n], el, ds, f"h{h} b{b}")
