"""Attention of a batch to a shared prefix on the GPU, alone, joined with either ring cache and
behind the batch's prompts, against 64 bits within the bounds of ``serving_reference``."""

from __future__ import annotations

import math

import pytest
import torch

import sbfa_native as native
from shared_prefix import SharedPrefix
from streaming_kv_cache import QuantizedStreamingKVCache, StreamingKVCache
from tests import serving_reference as ref
from tests.test_gpu_quantized_cache import check_attend, filled, gen, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(g, Hkv, P, D, dtype):
    return SharedPrefix(rows(g, (Hkv, P, D), dtype, 0.2), rows(g, (Hkv, P, D), dtype, 0.2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,G,N,P,D", [
    (1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 64, 128), (2, 2, 4, 1, 65, 128), (3, 1, 5, 7, 127, 80),
    (1, 2, 1, 127, 128, 64), (1, 1, 2, 64, 129, 128), (1, 3, 1, 129, 63, 40),
    (4, 2, 8, 8, 300, 96), (1, 1, 1, 257, 1000, 128), (2, 1, 3, 100, 2500, 72),
    (5, 2, 16, 1, 5000, 128), (64, 1, 8, 1, 777, 64),
])
def test_prefix_alone(dtype, B, Hkv, G, N, P, D):
    g = gen(20)
    pre = make(g, Hkv, P, D, dtype)
    q = rows(g, (B, N, Hkv * G, D), dtype, 0.3).transpose(1, 2)   # a view, as projections give
    o, lse = pre.attend(q, return_lse=True)
    u = ref.half_step(dtype)
    for h in range(Hkv):
        hs = slice(h * G, (h + 1) * G)
        eo, el, A, ds = ref.attention(q[:, hs].reshape(-1, D), pre.k[h], pre.v[h],
                                      1 / math.sqrt(D))
        ref.check(o[:, hs].reshape(-1, D), eo, A, ds, u, u, label=f"h{h}")
        ref.check_lse(lse[:, hs].reshape(-1), el, ds, f"h{h}")
    assert native.device_status() == 0


def test_prefix_scores_that_grow_along_it():
    """Maxima that keep growing make every row rescale, a softmax far from uniform."""
    g = gen(21)
    P, D = 1500, 128
    k = rows(g, (1, P, D), torch.bfloat16, 0.0)
    k += torch.linspace(-3, 3, P, device=DEV)[None, :, None].bfloat16()
    pre = SharedPrefix(k, rows(g, (1, P, D), torch.bfloat16, 0.5))
    q = (rows(g, (3, 4, 50, D), torch.bfloat16, 0.0) + 1).contiguous()
    o, lse = pre.attend(q, return_lse=True)
    eo, el, A, ds = ref.attention(q.reshape(-1, D), pre.k[0], pre.v[0], 1 / math.sqrt(D))
    u = 2.0 ** -8
    ref.check(o.reshape(-1, D), eo, A, ds, u, u)
    ref.check_lse(lse.reshape(-1), el, ds)


def test_a_nan_query_stays_alone():
    g = gen(22)
    pre = make(g, 1, 200, 64, torch.float16)
    q = rows(g, (2, 3, 70, 64), torch.float16)
    o = pre.attend(q)
    q[1, 2, 5] = math.nan
    bad = pre.attend(q)
    assert torch.isnan(bad[1, 2, 5]).all()
    bad[1, 2, 5] = o[1, 2, 5]
    assert torch.equal(bad, o)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16)])
@pytest.mark.parametrize("B,H,G,D,P,W,lengths", [
    (3, 2, 4, 128, 1000, 256, [0, 1, 900]), (2, 1, 1, 64, 1, 16, [0, 16]),
    (2, 3, 5, 80, 513, 33, [20, 0]), (9, 1, 17, 128, 130, 40, list(range(9)))])
def test_decode_behind_a_prefix(fmt, dtype, B, H, G, D, P, W, lengths):
    g = gen(23)
    c = filled(g, B, H, D, 0, W, dtype, fmt, lengths, 0.2)
    pre = make(g, H, P, D, dtype)
    check_attend(c, rows(g, (B, H * G, 1, D), dtype, 0.2), prefix=pre)
    assert native.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hkv,P,D", [(3, 300, 64), (1, 100, 128), (1, 9000, 128), (3, 1, 64)])
def test_decode_behind_a_prefix_with_the_16_bit_cache(dtype, Hkv, P, D):
    """One head per query head in the ring, fewer in the prefix; keys whole and cut into slices."""
    g = gen(24)
    B, H, S, W = 2, 3, 2, 50
    pre = make(g, Hkv, P, D, dtype)
    c = StreamingKVCache(B, H, D, S, W, dtype=dtype, device=DEV)
    k, v = (rows(g, (B, H, 90, D), dtype, 0.2) for _ in range(2))
    q = rows(g, (B, H, 1, D), dtype, 0.2)
    c.append(k, v)
    plain = c.attend(q)
    o, lse = c.attend(q, return_lse=True, prefix=pre)
    keep = ref.kept_positions(90, S, W)
    u = ref.half_step(dtype)
    for b in range(B):
        for h in range(H):
            p = h * Hkv // H
            eo, el, A, ds = ref.attention(q[b, h], torch.cat((pre.k[p], k[b, h, keep])),
                                          torch.cat((pre.v[p], v[b, h, keep])),
                                          1 / math.sqrt(D))
            # the own part is rounded once before the merge: u A more
            ref.check(o[b, h], eo, A, ds, u, 2 * u)
            ref.check_lse(lse[b, h], el, ds)
    assert torch.equal(c.attend(q), plain)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hkv,G,N,P,D,W", [
    (2, 2, 4, 100, 300, 128, 16), (1, 1, 1, 1, 1, 64, 1), (2, 1, 3, 33, 77, 80, 1000),
    (1, 2, 2, 300, 129, 64, 128),
    (37, 1, 2, 5, 200, 64, 3), (150, 2, 1, 1, 10, 128, 7), (9, 1, 5, 64, 128, 40, 20),
    (3, 1, 7, 65, 64, 96, 65), (2, 2, 1, 513, 5, 128, 200), (1, 1, 2, 700, 1500, 64, 701),
    (5, 1, 1, 129, 1000, 128, 129), (6, 1, 3, 8, 9000, 128, 8), (2, 1, 2, 300, 5000, 128, 300),
    (2, 1, 2, 600, 3333, 64, 500)])
def test_prompts_behind_a_prefix(dtype, B, Hkv, G, N, P, D, W):
    g = gen(25)
    pre = make(g, Hkv, P, D, dtype)
    q, k, v = (rows(g, (B, N, h, D), dtype, 0.2).transpose(1, 2) for h in (Hkv * G, Hkv, Hkv))
    o, lse = pre.attend_prompt(q, k, v, window_size=W, return_lse=True)
    i = torch.arange(N, device=DEV)
    gap = i[:, None] - i[None, :]
    seen = torch.cat((torch.ones(N, P, dtype=torch.bool, device=DEV), (gap >= 0) & (gap < W)), 1)
    u = ref.half_step(dtype)
    for b in range(B):
        for h in range(Hkv * G):
            kk = torch.cat((pre.k[h // G], k[b, h // G])).double()
            vv = torch.cat((pre.v[h // G], v[b, h // G])).double()
            x = (q[b, h].double() @ kk.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            w = torch.softmax(x, -1)
            ds = (q[b, h].double().abs() @ kk.abs().T).amax(-1) / math.sqrt(D) * D * 2.0 ** -23
            ref.check(o[b, h], w @ vv, w @ vv.abs(), ds, u, u)
            ref.check_lse(lse[b, h], torch.logsumexp(x, -1), ds)
    assert native.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,G,N,P,D,W", [(5, 3, 20, 100, 64, 7), (3, 2, 200, 40, 128, 30),
                                         (40, 1, 3, 3000, 80, 3), (2, 1, 90, 9000, 128, 50)])
def test_prompts_with_nan_and_infinities_in_some_rows(dtype, B, G, N, P, D, W):
    """Rows of one sequence do not reach another's, nor a query ahead of them (padding may hold
    anything); the queries that see them get what 64 bits give."""
    g = gen(30)
    pre = make(g, 1, P, D, dtype)
    q, k, v = (rows(g, (B, N, h, D), dtype, 0.2).transpose(1, 2) for h in (G, 1, 1))
    clean = pre.attend_prompt(q, k, v, window_size=W)
    k, v = k.clone(), v.clone()
    at = N // 2
    v[1, 0, at, 3], v[1, 0, at, D - 1] = math.nan, -math.inf      # seen by queries at .. at + W - 1
    v[1, 0, min(at + 1, N - 1), 5] = math.inf
    v[0, 0, N - 1, 2] = math.inf                                  # seen by the last query alone
    k[B - 1, 0, N - 1] = math.nan
    k[0, 0, N - 1, 0] = math.nan
    o = pre.attend_prompt(q, k, v, window_size=W)
    i = torch.arange(N, device=DEV)
    gap = i[:, None] - i[None, :]
    seen = (gap >= 0) & (gap < W)
    bad = ~torch.isfinite(v)
    for b in range(B):
        # a column is not finite where a seen value of it is not (or a seen key is NaN)
        col = (seen.double() @ bad[b, 0].double()) > 0
        row = (seen.double() @ (~torch.isfinite(k[b, 0]).all(-1)).double()) > 0
        want = (col | row[:, None]).expand(G, N, D)
        assert torch.equal(~torch.isfinite(o[b]), want), b
        assert torch.equal(o[b][~want], clean[b][~want]), b
    one = o[1, :, at, D - 1]
    assert torch.equal(one, torch.full_like(one, -math.inf))
    assert torch.isnan(o[1, :, at, 3]).all()
    assert native.device_status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_serving_run(fmt):
    """Shared system prompt, ragged prompts, decode steps, then the cache handed over: each step
    against attention over everything the sequence may see."""
    g = gen(26)
    B, H, G, D, P, W, N = 3, 2, 4, 128, 200, 40, 64
    dt = torch.bfloat16
    pre = make(g, H, P, D, dt)
    cache = QuantizedStreamingKVCache(B, H, D, 0, W, dtype=dt, fmt=fmt, device=DEV)
    counts = torch.tensor([0, 17, N], device=DEV)
    k, v = (rows(g, (B, H, N + 30, D), dt, 0.2) for _ in range(2))
    q = rows(g, (B, H * G, N, D), dt, 0.2)
    o = pre.attend_prompt(q, k[:, :, :N], v[:, :, :N], window_size=W)
    alone = pre.attend_prompt(q[1:2, :, :17], k[1:2, :, :17], v[1:2, :, :17], window_size=W)
    # padding changes nothing but the split of the sums: two weight and two output roundings
    assert (o[1:2, :, :17].double() - alone.double()).abs().max() <= 4 * 2.0 ** -8 * 8
    cache.append(k[:, :, :N], v[:, :, :N], counts)
    seqs = [[(k[b, :, t], v[b, :, t]) for t in range(int(counts[b]))] for b in range(B)]
    for t in range(N, N + 30):
        cache.append(k[:, :, t:t + 1], v[:, :, t:t + 1])
        for b in range(B):
            seqs[b].append((k[b, :, t], v[b, :, t]))
        check_attend(cache, rows(g, (B, H * G, 1, D), dt, 0.2), prefix=pre, label=f"t{t}")
    assert cache.lengths.tolist() == [len(s) for s in seqs]
    kr, vr, pos = cache.read()
    for b, s in enumerate(seqs):
        keep = [p for p in pos[b].tolist() if p >= 0]
        assert keep == list(range(max(0, len(s) - W), len(s)))
        for got, part in ((kr, 0), (vr, 1)):
            want = torch.stack([s[p][part] for p in keep], 1).double()
            # one rounding of a code: half a step of it (e4m3: 2^-4 of the value, or of the
            # smallest normal code; int8: half a code), scales at most twice the smallest
            amax = want.abs().amax(-1, keepdim=True)
            tol = (torch.maximum(want.abs() * 2.0 ** -4, amax * 2.0 ** -9 / 448 * 2)
                   if fmt == "e4m3" else amax / 127 * 2 / 2)
            assert ((got[b, :, :len(keep)].double() - want).abs() <= tol).all()
    assert native.device_status() == 0


def test_captured_and_replayed():
    g = gen(27)
    B, H, G, D, P = 2, 2, 4, 64, 500
    pre = make(g, H, P, D, torch.bfloat16)
    cache = filled(g, B, H, D, 0, 64, torch.bfloat16, "e4m3", [5, 70])
    q = rows(g, (B, H * G, 1, D), torch.bfloat16)
    qp, kp, vp = (rows(g, (B, h, 40, D), torch.bfloat16) for h in (H * G, H, H))
    want = cache.attend(q, prefix=pre), pre.attend_prompt(qp, kp, vp, window_size=16)
    graphs = []
    for _ in range(2):   # two graphs of the same call, replayed at the same time
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            out = cache.attend(q, prefix=pre), pre.attend_prompt(qp, kp, vp, window_size=16)
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(20):
        for graph, _, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for _, out, s in graphs:
            torch.cuda.current_stream().wait_stream(s)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_many_sequences_behind_a_prefix_on_two_streams():
    """Several waves of prefix CTAs beside a cache cut into equal runs, twice at the same time."""
    g = gen(31)
    B, H, G, D, P, W = 700, 2, 4, 64, 260, 2500
    pre = make(g, H, P, D, torch.float16)
    c = filled(g, 4, H, D, 0, W, torch.float16, "int8", [0, 7, 2500, 9000])
    big = QuantizedStreamingKVCache(B, H, D, 0, W, dtype=torch.float16, fmt="int8", device=DEV)
    pick = torch.arange(B, device=DEV) % 4
    big.load(c.k[pick], c.v[pick], c.scales[pick], c.lengths[pick])
    qs = [rows(g, (4, H * G, 1, D), torch.float16, 0.2) for _ in range(2)]
    want = [check_attend(c, q, prefix=pre) for q in qs]
    outs = [big.attend(q[pick], return_lse=True, prefix=pre) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    again = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                again[i].append(big.attend(qs[i][pick], return_lse=True, prefix=pre))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i in range(2):
        # the same sums in another split: within the output's rounding and the weights'
        tol = 4 * 2.0 ** -11 * want[i][0].double().abs().amax() + 1e-30
        assert ((outs[i][0].double() - want[i][0][pick].double()).abs() <= tol).all()
        assert ((outs[i][1] - want[i][1][pick]).abs() <= 1e-4 * (1 + want[i][1][pick].abs())).all()
        assert all(torch.equal(a, b) for o in again[i] for a, b in zip(o, outs[i]))
    assert native.device_status() == 0


def test_prefix_copies_only_what_it_must():
    g = gen(28)
    k = rows(g, (2, 50, 64), torch.float16)
    t = rows(g, (50, 2, 64), torch.float16).transpose(0, 1)
    pre = SharedPrefix(k, t)
    assert pre.k.data_ptr() == k.data_ptr() and pre.v.is_contiguous()
    q = rows(g, (1, 2, 3, 64), torch.float16)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(pre.attend(q), pre.attend(odd))
    wide = q[:, :1].expand(1, 2, 3, 64)
    assert torch.equal(pre.attend(wide), pre.attend(wide.contiguous()))
    kv = rows(g, (1, 1, 3, 64), torch.float16).expand(1, 2, 3, 64)   # a stride of zero
    oddk = torch.empty(kv.numel() + 1, dtype=kv.dtype, device=DEV)[1:].view(kv.shape)
    oddk.copy_(kv)
    want = pre.attend_prompt(q, kv.contiguous(), kv.contiguous(), 2)
    assert torch.equal(want, pre.attend_prompt(odd, kv, oddk, 2))


def test_refusals():
    g = gen(29)
    pre = make(g, 2, 50, 64, torch.float16)
    q = rows(g, (2, 4, 3, 64), torch.float16)
    k = rows(g, (2, 2, 3, 64), torch.float16)
    for bad in (lambda: pre.attend(q[:, :3]), lambda: pre.attend(q[..., :32]),
                lambda: pre.attend(q.bfloat16()), lambda: pre.attend(q.cpu()),
                lambda: pre.attend(q[:, :, :0]), lambda: pre.attend(q[0]),
                lambda: pre.attend_prompt(q, k[:, :1], k[:, :1], 4),
                lambda: pre.attend_prompt(q, k, k[:, :, :2], 4),
                lambda: pre.attend_prompt(q, k, k, 0),
                lambda: pre.attend_prompt(q, k.bfloat16(), k.bfloat16(), 4),
                lambda: SharedPrefix(k[0], k[0].bfloat16()),
                lambda: SharedPrefix(k[0].float(), k[0].float()),
                lambda: SharedPrefix(k[0][..., :60], k[0][..., :60])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="softmax_scale"):
        pre.attend(q, softmax_scale=-1.0)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        pre.attend_prompt(q, k, k, 4, softmax_scale=0.0)
    with pytest.raises(RuntimeError, match="gradients"):
        pre.attend(q.clone().requires_grad_(True))
    c = filled(g, 2, 2, 64, 0, 8, torch.bfloat16, "int8", [3, 4])
    with pytest.raises(ValueError, match="the cache"):
        c.attend(q[:, :, :1].bfloat16(), prefix=pre)
    c = filled(g, 2, 1, 64, 0, 8, torch.float16, "int8", [3, 4])
    with pytest.raises(ValueError, match="the cache"):
        c.attend(q[:, :, :1], prefix=pre)
    f32 = StreamingKVCache(1, 2, 64, 0, 8, dtype=torch.float32, device=DEV)
    f32.append(torch.zeros(1, 2, 1, 64, device=DEV), torch.zeros(1, 2, 1, 64, device=DEV))
    with pytest.raises(ValueError, match="q must be"):
        f32.attend(torch.zeros(1, 2, 1, 64, device=DEV), prefix=pre)
