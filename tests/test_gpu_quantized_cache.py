"""The 8-bit ring cache on the GPU: codes, scales and lengths equal the definition's bit for bit,
attention holds the bounds of ``serving_reference``, reading back is exact."""

from __future__ import annotations

import math

import pytest
import torch

import sbfa_native as native
from streaming_kv_cache import QuantizedStreamingKVCache as Cache
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(g, shape, dtype, spread=0.5):
    x = torch.randn(shape, generator=g, device=DEV)
    return (x * torch.exp(spread * torch.randn(shape[:-1], generator=g, device=DEV))[..., None]
            ).to(dtype)


def filled(g, B, H, D, S, W, dtype, fmt, lengths, spread=0.5):
    """A cache whose every ring row holds quantised values, whatever the lengths say."""
    c = Cache(B, H, D, S, W, dtype=dtype, fmt=fmt, device=DEV)
    code_dtype = c.k.dtype
    kc, kb = ref.quantise(rows(g, (B, H, S + W, D), dtype, spread), fmt)
    vc, vb = ref.quantise(rows(g, (B, H, S + W, D), dtype, spread), fmt)
    c.load(kc.to(code_dtype), vc.to(code_dtype), torch.stack((kb, vb), -1),
           torch.tensor(lengths, dtype=torch.int64, device=DEV))
    return c


def state(c):
    return c.k.double(), c.v.double(), c.scales.clone(), c.lengths.clone()


def expect_append(st, k, v, counts, S, W, fmt):
    """The state after an append, row by row."""
    ek, ev, es, el = st
    for part, (x, held) in enumerate(((k, ek), (v, ev))):
        codes, byte = ref.quantise(x, fmt)
        for b, n in enumerate(counts):
            L = int(st[3][b])
            for t in range(n):
                p = L + t
                if p >= S and p < L + n - W:
                    continue
                r = ref.ring_row(p, S, W)
                held[b, :, r] = codes[b, :, t]
                es[b, :, r, part] = byte[b, :, t]
    return ek, ev, es, el + torch.tensor(counts, device=DEV)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,B,H,D,S,W,lengths,T,counts", [
    (torch.bfloat16, 2, 3, 128, 4, 29, [0, 7], 1, None),
    (torch.float16, 3, 1, 64, 4, 29, [0, 3, 100], 70, [0, 70, 33]),
    (torch.bfloat16, 1, 5, 80, 0, 16, [5], 40, None),
    (torch.float16, 2, 2, 256, 3, 0, [0, 2], 9, None),
    (torch.bfloat16, 4, 2, 40, 1, 7, [0, 1, 8, 9], 8, [8, 1, 0, 5]),
    (torch.float16, 1, 1, 8, 2, 300, [290], 700, None),
])
def test_append_writes_the_definition(fmt, dtype, B, H, D, S, W, lengths, T, counts):
    g = gen(1)
    c = filled(g, B, H, D, S, W, dtype, fmt, lengths)
    # [B, T, H, D] storage seen as [B, H, T, D], as projections leave it
    k = rows(g, (B, T, H, D), dtype).transpose(1, 2)
    v = rows(g, (B, T, H, D), dtype).transpose(1, 2)
    want = expect_append(state(c), k, v, counts or [T] * B, S, W, fmt)
    c.append(k, v, None if counts is None else torch.tensor(counts, device=DEV))
    for got, exp in zip(state(c), want):
        assert torch.equal(got, exp)
    assert not c._tickets.any() and not c._k[..., D:].any() and not c._v[..., D:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_special_rows(fmt, dtype):
    """Zeros, the type's extremes and subnormals, ties between codes, NaN and infinities."""
    fi = torch.finfo(dtype)
    D = 64
    x = torch.zeros(12, D, device=DEV)
    x[1] = fi.max
    x[2, 3] = fi.smallest_normal
    x[3, 5] = fi.smallest_normal * fi.eps        # the smallest subnormal
    x[4] = torch.linspace(-fi.max / 2, fi.max / 2, D, device=DEV)
    x[5, 0], x[5, 1:] = 127.0, torch.arange(1, D, device=DEV) / 2.0     # int8 ties
    x[6, 0], x[6, 1:] = 448.0, 16.5 + torch.arange(D - 1, device=DEV)   # e4m3 ties
    x[7, 0] = 448.0 * 2 ** 5
    x[8, 0] = 127.0 * 2 ** 5
    x[9, 1] = math.inf
    x[10, 2] = -math.inf
    x[11, 3] = math.nan
    x = x.to(dtype)[None, None]
    c = Cache(1, 1, D, 0, 16, dtype=dtype, fmt=fmt, device=DEV)
    c.append(x, x.flip(2))
    for codes, part, src in ((c.k, 0, x), (c.v, 1, x.flip(2))):
        want, byte = ref.quantise(src, fmt)
        assert torch.equal(codes[:, :, :12].double(), want)
        assert torch.equal(c.scales[:, :, :12, part], byte)
    kr, vr, pos = c.read()
    assert torch.equal(pos[0], torch.tensor(list(range(12)) + [-1] * 4, device=DEV))
    assert torch.isnan(kr[0, 0, 9:12]).all() and torch.isfinite(kr[0, 0, :9]).all()
    assert torch.isnan(vr[0, 0, 0:3]).all() and not kr[0, 0, 12:].any()
    # the largest value of the type rounds up to a code past it and saturates
    c.reset()
    c.append(torch.zeros_like(x[:, :, :1]), x[:, :, 1:2])
    o = c.attend(torch.ones_like(x[:, :, :1]))
    assert torch.equal(o, torch.full_like(o, fi.max)) and torch.equal(c.read()[1][:, :, :1], o)


def test_append_counts_are_clamped_and_padding_is_not_read():
    g = gen(2)
    c = Cache(3, 2, 64, 2, 8, fmt="int8", device=DEV)
    k = rows(g, (3, 2, 5, 64), torch.bfloat16)
    k[0] = math.nan
    k[2, :, 3:] = math.inf
    c.append(k, k, torch.tensor([-4, 99, 3], device=DEV))
    assert c.lengths.tolist() == [0, 5, 3]
    kr, vr, pos = c.read()
    assert torch.isfinite(kr).all() and torch.isfinite(vr).all()
    assert pos[2].tolist() == [0, 1, 2] + [-1] * 7


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16)])
@pytest.mark.parametrize("B,H,D,S,W,lengths", [
    (5, 2, 128, 4, 33, [0, 1, 37, 38, 1000]), (2, 3, 40, 0, 5, [3, 77]),
    (2, 1, 256, 7, 0, [3, 50]), (1, 1, 64, 3, 1000, [10 ** 12 + 7])])
def test_read_gives_the_kept_positions_in_order(fmt, dtype, B, H, D, S, W, lengths):
    c = filled(gen(3), B, H, D, S, W, dtype, fmt, lengths)
    k, v, pos = c.read()
    for b, L in enumerate(lengths):
        lo = list(range(min(L, S)))
        keep = lo + list(range(max(S, L - W), L)) if L > S else lo
        assert pos[b].tolist() == keep + [-1] * (S + W - len(keep))
        at = [ref.ring_row(p, S, W) for p in keep]
        for h in range(H):
            fk, fv = ref.values(c, b, h)
            for got, full in ((k, fk), (v, fv)):
                assert torch.equal(got[b, h, :len(at)], full[at].to(dtype))
                assert not got[b, h, len(at):].any()


def check_attend(c, q, scale=None, prefix=None, label=""):
    B, Hq, _, D = q.shape
    G = Hq // c.heads
    sc = 1 / math.sqrt(D) if scale is None else scale
    o, lse = c.attend(q, scale, return_lse=True, prefix=prefix)
    u = ref.half_step(c.dtype)
    for b in range(B):
        n = min(int(c.lengths[b]), c.sink_size + c.window_size)
        for h in range(c.heads):
            k, v = (x[:n] for x in ref.values(c, b, h))
            big = v.abs().max().item() if n else 0.0
            u_p = ref.U16
            if prefix is not None:
                k = torch.cat((prefix.k[h].double(), k))
                v = torch.cat((prefix.v[h].double(), v))
                u_p = max(u_p, u)
            hs = slice(h * G, (h + 1) * G)
            eo, el, A, ds = ref.attention(q[b, hs, 0], k, v, sc)
            ref.check(o[b, hs, 0], eo, A, ds, u, u_p, n * 2.0 ** -25 * big, f"{label} b{b} h{h}")
            if k.shape[0] == 0:
                assert not o[b, hs].any() and not lse[b, hs].any()
            else:
                ref.check_lse(lse[b, hs, 0], el, ds, f"{label} b{b} h{h}")
    return o, lse


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.bfloat16),
                                       ("e4m3", torch.float16), ("int8", torch.float16)])
@pytest.mark.parametrize("B,H,G,D,S,W,lengths", [
    (3, 2, 4, 128, 4, 1000, [0, 1, 5000]),
    (1, 1, 1, 64, 0, 16, [16]),
    (4, 3, 5, 80, 3, 77, [15, 16, 17, 33]),
    (2, 1, 8, 256, 4, 130, [131, 500]),
    (2, 2, 12, 128, 1, 64, [2, 64]),
    (1, 2, 16, 64, 4, 300, [257]),
    (2, 1, 17, 96, 4, 50, [54, 9]),
    (1, 1, 33, 256, 0, 40, [39]),
    (40, 8, 2, 128, 0, 40, list(range(40))),
    # many units: equal runs of steps over all of them
    (64, 2, 4, 128, 4, 500, [(b * 37) % 600 for b in range(64)]),
    (200, 2, 1, 64, 0, 33, [b % 36 for b in range(200)]),
    (20, 6, 12, 80, 2, 300, [0] * 7 + [302] + [0] * 4 + [1, 500, 31, 32, 33, 64, 65, 0]),
    (37, 3, 9, 256, 4, 90, [b * 5 for b in range(37)]),
    (300, 1, 17, 64, 0, 20, [3] * 300),
    (130, 1, 2, 128, 0, 16, [0] * 130),
    (7, 16, 1, 128, 0, 9000, [9000, 0, 8999, 1, 4500, 12, 7]),
])
def test_attend_matches_64_bits(fmt, dtype, B, H, G, D, S, W, lengths):
    g = gen(4)
    c = filled(g, B, H, D, S, W, dtype, fmt, lengths)
    q = rows(g, (B, H * G, 1, D), dtype)
    check_attend(c, q)
    assert native.device_status() == 0


@pytest.mark.parametrize("H", [1, 3])
def test_attend_every_length_of_a_short_ring(H):
    S, W = 2, 70
    lengths = list(range(74))
    g = gen(5)
    c = filled(g, len(lengths), H, 64, S, W, torch.bfloat16, "int8", lengths)
    check_attend(c, rows(g, (len(lengths), 3 * H, 1, 64), torch.bfloat16), scale=0.3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_rows_of_very_different_magnitude(dtype):
    """Value rows from 2^-14 to 2^14, zero rows among them, and scores that grow along the cache: the
    references of the weights and of the row sum move apart."""
    g = gen(6)
    B, H, D, n = 2, 2, 128, 500
    c = Cache(B, H, D, 4, 996, dtype=dtype, device=DEV)
    k = torch.randn(B, H, n, D, generator=g, device=DEV) * torch.linspace(0.1, 3, n, device=DEV)[
        :, None]
    v = torch.randn(B, H, n, D, generator=g, device=DEV)
    v *= torch.exp2(torch.randint(-14, 13, (B, H, n, 1), generator=g, device=DEV).float())
    v[:, :, ::7] = 0
    c.append(k.to(dtype), v.to(dtype))
    check_attend(c, rows(g, (B, H * 4, 1, D), dtype))


def test_attend_queries_outside_fp16():
    """bf16 queries far above and below fp16's range, against keys that bring the scores back."""
    g = gen(7)
    D, n = 64, 90
    c = Cache(1, 1, D, 0, 100, device=DEV)
    k = torch.randn(1, 1, n, D, generator=g, device=DEV)
    q = torch.randn(1, 3, 1, D, generator=g, device=DEV)
    up = torch.tensor([2.0 ** 40, 1.0, 2.0 ** -60], device=DEV)[None, :, None, None]
    c.append((k * 2.0 ** -40).bfloat16(), k.bfloat16())
    check_attend(c, (q * up).bfloat16(), label="small keys")
    c.reset()
    c.append((k * 2.0 ** 60).bfloat16(), k.bfloat16())
    check_attend(c, (q[:, 2:] * 2.0 ** -60).bfloat16(), label="large keys")


def test_attend_does_not_see_what_lies_behind_the_length():
    g = gen(8)
    B, H, D, S, W = 2, 2, 128, 4, 60
    c = filled(g, B, H, D, S, W, torch.bfloat16, "e4m3", [33, 20])
    q = rows(g, (B, 2 * H, 1, D), torch.bfloat16)
    o = c.attend(q)
    c.scales[0, :, 33:] = 255
    c.scales[1, :, 20:] = 255
    assert torch.equal(c.attend(q), o)
    # ... and a NaN row that it does see reaches its own heads alone
    c.scales[0, 1, 5, 1] = 255
    bad = c.attend(q)
    assert torch.isnan(bad[0, 2:]).all()
    assert torch.equal(bad[0, :2], o[0, :2]) and torch.equal(bad[1], o[1])
    c.scales[0, 1, 5, 1] = 120
    c.scales[0, 1, 5, 0] = 255
    assert torch.isnan(c.attend(q)[0, 2:]).all()


def test_attend_heads_of_a_group_are_independent():
    """A NaN query makes its own row NaN and no other."""
    g = gen(9)
    c = filled(g, 1, 1, 128, 0, 200, torch.float16, "int8", [150])
    q = rows(g, (1, 8, 1, 128), torch.float16)
    o = c.attend(q)
    q[0, 3] = math.nan
    bad = c.attend(q)
    assert torch.isnan(bad[0, 3]).all()
    keep = [i for i in range(8) if i != 3]
    assert torch.equal(bad[0, keep], o[0, keep])


def test_views_and_misaligned_inputs():
    g = gen(10)
    B, H, D, T = 2, 2, 64, 9
    base = rows(g, (B, T, 3, H, D), torch.bfloat16)          # packed q, k, v
    k, v = base[:, :, 1].transpose(1, 2), base[:, :, 2].transpose(1, 2)
    odd = torch.empty(B * H * T * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(B, H, T, D)
    odd.copy_(k)
    one = k[:, :1].expand(B, H, T, D)                         # a stride of zero
    caches = [Cache(B, H, D, 1, 20, device=DEV) for _ in range(4)]
    caches[0].append(k, v)
    caches[1].append(odd, v.contiguous())
    assert torch.equal(caches[0]._k, caches[1]._k) and torch.equal(caches[0]._v, caches[1]._v)
    caches[2].append(one, v)
    caches[3].append(one.contiguous(), v)
    assert torch.equal(caches[2]._k, caches[3]._k)
    q = torch.empty(B * H * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(B, H, 1, D)
    q.copy_(base[:, :1, 0].transpose(1, 2))
    assert torch.equal(caches[0].attend(q), caches[0].attend(base[:, :1, 0].transpose(1, 2)))


def test_step_captured_and_replayed_advances():
    g = gen(11)
    B, H, G, D, S, W = 3, 2, 4, 128, 4, 24
    a, b = (Cache(B, H, D, S, W, device=DEV) for _ in range(2))
    k = rows(g, (B, H, 50, D), torch.bfloat16)
    q = rows(g, (50, B, H * G, 1, D), torch.bfloat16)
    first = torch.tensor([0, 3, 9], device=DEV)
    for c in (a, b):
        c.append(k[:, :, :9], k[:, :, :9], first)
    ks, qs = k[:, :, :1].clone(), q[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Cache(B, H, D, S, W, device=DEV).attend(qs)     # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        a.append(ks, ks)
        og = a.attend(qs)
    for t in range(9, 50):
        ks.copy_(k[:, :, t:t + 1])
        qs.copy_(q[t])
        graph.replay()
        b.append(k[:, :, t:t + 1], k[:, :, t:t + 1])
        assert torch.equal(og, b.attend(q[t]))
    assert torch.equal(a.lengths, first + 41) and torch.equal(a._k, b._k)


def test_other_stream_and_state_round_trip():
    g = gen(12)
    c = filled(g, 2, 2, 64, 4, 60, torch.float16, "int8", [10, 100])
    q = rows(g, (2, 4, 1, 64), torch.float16)
    o = c.attend(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2 = c.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2)
    d = Cache(2, 2, 64, 4, 60, dtype=torch.float16, fmt="int8", device=DEV)
    d.load(c.k, c.v, c.scales, c.lengths)
    assert torch.equal(d.attend(q), o)
    d.reset([1])
    assert d.lengths.tolist() == [10, 0] and not d.attend(q)[1].any()
    d.reset()
    assert not d.lengths.any()


def test_offsets_beyond_32_bits():
    """One head of 2^25 + 9 rows of 128 bytes: its last rows lie behind 2^32 bytes."""
    D, n = 128, 2 ** 25 + 9
    c = Cache(1, 1, D, 0, n, device=DEV)
    one = torch.zeros(1, 1, 1, D, dtype=torch.bfloat16, device=DEV)
    c.lengths.fill_(n - 1)
    key, val = one.clone(), one.clone()
    key[..., 0], val[...] = 64.0, torch.arange(D, device=DEV) % 8
    c.append(key, val)                      # row n - 1
    assert int(c.lengths[0]) == n
    assert torch.equal(c.v[0, 0, n - 1].float(), (torch.arange(D, device=DEV) % 8) * 64.0)
    q = one.clone()
    q[..., 0] = 8.0
    # scores: 512 for the last row, 0 for the zero rows, whose weight vanishes
    o, lse = c.attend(q, softmax_scale=1.0, return_lse=True)
    assert torch.equal(o[0, 0, 0], val[0, 0, 0])
    assert abs(lse.item() - 512.0) <= 2.0 ** -17 * 513
    # equal scores: the mean of all rows
    o, lse = c.attend(one, softmax_scale=1.0, return_lse=True)
    assert abs(lse.item() - math.log(n)) <= 2.0 ** -15 * math.log(n)
    want = val[0, 0, 0].double() / n
    assert ((o[0, 0, 0].double() - want).abs() <= 2.0 ** -7 * want).all()


@pytest.mark.parametrize("B,H,G,W,top", [(65535, 1, 1, 9, 12), (3000, 3, 2, 40, 90),
                                         (1, 70000, 1, 5, 4), (2, 300, 9, 33, 30)])
def test_many_sequences_and_heads(B, H, G, W, top):
    """Grids at their limits: every sequence's length, and a sample of the results."""
    g = gen(13)
    D = 64
    c = Cache(B, H, D, 1, W, fmt="int8", device=DEV)
    k, v = (torch.randn(B, H, 2, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    c.append(k, v)
    assert (c.lengths == 2).all() and not c._tickets.any()
    c._k.random_(0, 255, generator=g)
    c._v.random_(0, 255, generator=g)
    c.scales.random_(118, 124, generator=g)
    c.lengths.random_(0, top + 1, generator=g)
    q = torch.randn(B, H * G, 1, D, generator=g, device=DEV).bfloat16()
    o, lse = c.attend(q, return_lse=True)
    empty = c.lengths == 0
    assert not o[empty].any() and not lse[empty].any()
    assert (lse[~empty] != 0).all() and torch.isfinite(o).all()
    for b, h in {(0, 0), (B - 1, H - 1), (B // 2, H // 3), (B // 3, H // 2), (B - 1, 0)}:
        n = min(int(c.lengths[b]), 1 + W)
        kk, vv = (x[:n] for x in ref.values(c, b, h))
        hs = slice(h * G, (h + 1) * G)
        eo, _, A, ds = ref.attention(q[b, hs, 0], kk, vv, 1 / math.sqrt(D))
        big = vv.abs().max().item() if n else 0.0
        ref.check(o[b, hs, 0], eo, A, ds, 2.0 ** -8, ref.U16, n * 2.0 ** -25 * big, f"b{b} h{h}")


def test_two_attends_at_the_same_time():
    g = gen(14)
    c = filled(g, 32, 8, 128, 4, 1500, torch.bfloat16, "e4m3", [b * 50 for b in range(32)])
    qs = [rows(g, (32, 32, 1, 128), torch.bfloat16) for _ in range(2)]
    want = [c.attend(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(c.attend(qs[i]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_refusals():
    c = Cache(2, 2, 64, 4, 12, device=DEV)
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: c.append(x[:, :1], x[:, :1]), lambda: c.append(x, x[:, :, :2]),
                lambda: c.append(x.half(), x.half()), lambda: c.append(x.cpu(), x.cpu()),
                lambda: c.append(x[0], x[0]),
                lambda: c.append(x, x, torch.zeros(3, dtype=torch.int64, device=DEV)),
                lambda: c.append(x, x, torch.zeros(2, device=DEV)),
                lambda: c.append(x, x, torch.zeros(2, dtype=torch.int64)),
                lambda: c.attend(q[:, :3]), lambda: c.attend(q[:1]), lambda: c.attend(x),
                lambda: c.attend(q[:, :0]), lambda: c.attend(q.half()),
                lambda: c.load(c.k, c.v, c.scales, c.lengths - 1),
                lambda: c.load(c.k, c.v, c.scales, c.lengths.int()),
                lambda: c.load(c.k[:1], c.v, c.scales, c.lengths),
                lambda: c.load(c.k.view(torch.int8), c.v, c.scales, c.lengths)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="softmax_scale"):
        c.attend(q, softmax_scale=-1.0)
    with pytest.raises(RuntimeError, match="gradients"):
        c.attend(q.requires_grad_(True))
    with torch.no_grad():
        assert not c.attend(q).any()
    with pytest.raises(AttributeError):
        c.lengths = c.lengths + 1
    c.append(x[:, :, :0], x[:, :, :0])
    assert not c.lengths.any()
