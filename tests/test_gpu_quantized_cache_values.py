"""Attention over the 8-bit ring where one value row must not decide how finely the others are
weighed: rows of zeros (an attention sink, a padding token) and rows that are large in one column.
In every form of the kernel: a cluster per unit, equal runs, behind a prefix.  And scores that are
all minus infinity."""

from __future__ import annotations

import math

import pytest
import torch

import sbfa_native as native
from shared_prefix import SharedPrefix
from streaming_kv_cache import QuantizedStreamingKVCache as Cache
from tests import serving_reference as ref
from tests.test_gpu_quantized_cache import gen, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOG2 = math.log(2.0)   # as softmax_scale: scores count powers of two
TYPES = [("e4m3", torch.bfloat16), ("int8", torch.bfloat16), ("e4m3", torch.float16),
         ("int8", torch.float16)]
# heads, rows, grouped queries; 36 sequences of these make a cluster's units and equal runs
FORMS = {"cluster": (1, 1000, 4), "two sets": (1, 1000, 12), "runs": (4, 6000, 2),
         "prefix": (1, 1000, 4)}


def keys_and_queries(g, B, H, G, n, D, dtype):
    """Scores (in powers of two) of about 0 each, as long as column 0 of the keys is 0; what stands
    there adds 4 times itself."""
    k = 0.05 * torch.randn(B, H, n, D, generator=g, device=DEV)
    q = 0.25 * torch.randn(B, H * G, 1, D, generator=g, device=DEV)
    k[..., 0], q[..., 0] = 0.0, 4.0
    return k, q.to(dtype)


def cache_of(form, B, D, dtype, fmt):
    H, n, G = FORMS[form]
    c = Cache(B, H, D, 4, n - 4, dtype=dtype, fmt=fmt, device=DEV)
    need = native.lib().sbfa_qcache_attend_workspace_bytes(c._handle, H * G)
    assert (need > 0) == (form == "runs")
    prefix = None
    if form == "prefix":   # far below the own scores: the cache's part decides
        g = gen(42)
        kp = torch.zeros(H, 70, D, device=DEV)
        kp[..., 0] = -5.0
        vp = 2.0 ** -14 * torch.randn(H, 70, D, generator=g, device=DEV)
        prefix = SharedPrefix(kp.to(dtype), vp.to(dtype))
    return c, H, n, G, prefix


def check_attend(c, q, prefix=None):
    """Every sequence and head within the bound of ``serving_reference.check`` and half a step of the
    output type's subnormals: outputs below fp16's 2^-14 are rounded to multiples of 2^-24, off by up
    to 2^-25 whatever their size (bf16: 2^-134)."""
    B, Hq, _, _ = q.shape
    G = Hq // c.heads
    o, lse = c.attend(q, LOG2, return_lse=True, prefix=prefix)
    fi = torch.finfo(c.dtype)
    u = ref.half_step(c.dtype)
    for b in range(B):
        n = min(int(c.lengths[b]), c.sink_size + c.window_size)
        for h in range(c.heads):
            k, v = (x[:n] for x in ref.values(c, b, h))
            extra = n * 2.0 ** -25 * v.abs().max().item() + fi.smallest_normal * fi.eps / 2
            u_p = ref.U16
            if prefix is not None:
                k = torch.cat((prefix.k[h].double(), k))
                v = torch.cat((prefix.v[h].double(), v))
                u_p = max(u_p, u)
            hs = slice(h * G, (h + 1) * G)
            eo, el, A, ds = ref.attention(q[b, hs, 0], k, v, LOG2)
            ref.check(o[b, hs, 0], eo, A, ds, u, u_p, extra, f"b{b} h{h}")
            ref.check_lse(lse[b, hs, 0], el, ds, f"b{b} h{h}")
    return o, lse


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("form,D", [(f, d) for f in FORMS for d in (64, 128)
                                    if (f, d) != ("runs", 64)] + [("cluster", 256)])
def test_a_zero_value_row_does_not_coarsen_the_others(form, D, fmt, dtype):
    """One zero row per sequence, first, last or alone in its warp's share, its score 0, 6 or 10
    powers of two above the others', among values of 1 down to 2^-14."""
    g = gen(40)
    cases = [(amp, lead, at) for amp in (0, -5, -10, -14) for lead in (0, 6, 10)
             for at in ("first", "last", "alone")]
    B = len(cases)
    c, H, n, G, prefix = cache_of(form, B, D, dtype, fmt)
    k, q = keys_and_queries(g, B, H, G, n, D, dtype)
    v = 1 + 0.5 * torch.randn(B, H, n, D, generator=g, device=DEV)
    counts = []
    for b, (amp, lead, at) in enumerate(cases):
        counts.append(33 if at == "alone" else n - b % 3)
        row = 0 if at == "first" else counts[-1] - 1
        v[b] *= 2.0 ** amp
        v[b, :, row] = 0.0
        v[b, :, row, ::2] = -0.0
        k[b, :, row, 0] = lead / 4
    c.append(k.to(dtype), v.to(dtype), torch.tensor(counts, device=DEV))
    assert (c.scales[0, :, 0, 1] == 127).all()
    check_attend(c, q, prefix)


@pytest.mark.parametrize("fmt,dtype", TYPES)
def test_zero_rows_beside_rows_of_the_same_scale_byte(fmt, dtype):
    """Values of a few hundred have the scale byte of a zero row; zero rows only, none, or a NaN row
    among them."""
    g = gen(43)
    D, n = 128, 300
    c = Cache(4, 2, D, 0, n, dtype=dtype, fmt=fmt, device=DEV)
    k, q = keys_and_queries(g, 4, 2, 4, n, D, dtype)
    v = torch.randn(4, 2, n, D, generator=g, device=DEV).clamp(-1, 1) * ref.TOP[fmt] / 4
    v[..., 7] = ref.TOP[fmt]
    v[1] = 0.0
    v[2, :, ::5] = 0.0
    v[3, :, 1:] = 0.0
    c.append(k.to(dtype), v.to(dtype))
    assert (c.scales[..., 1] == 127).all()
    o, lse = check_attend(c, q)
    assert not o[1].any()
    c.scales[2, 1, 10, 1] = 255
    bad, bad_lse = c.attend(q, LOG2, return_lse=True)
    assert torch.isnan(bad[2, 4:]).all() and torch.equal(bad_lse, lse)
    bad[2, 4:] = o[2, 4:]
    assert torch.equal(bad, o)


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_a_row_large_in_one_column_does_not_coarsen_the_others(form, fmt, dtype):
    """The first row holds 2^10 in one column, zeros in the others, and a score 14 powers of two above
    the rest: the other columns come from the other rows alone.

    Bound: the kernel's reference M of the weighted values lies at least 11 powers of two below
    the largest weight times scale, so a weight that falls below fp16's normal range is off by at most
    2^-25 2^M <= 2^-36 max_i(w_i 2^e_i) for each code of the column."""
    g = gen(44)
    B, D = 36, 128
    c, H, n, G, prefix = cache_of(form, B, D, dtype, fmt)
    k, q = keys_and_queries(g, B, H, G, n, D, dtype)
    v = 1 + 0.5 * torch.randn(B, H, n, D, generator=g, device=DEV)
    v[:, :, 0], k[:, :, 0, 0] = 0.0, 14 / 4
    v[:, :, 0, 17] = 2.0 ** 10
    c.append(k.to(dtype), v.to(dtype))
    o = c.attend(q, LOG2, prefix=prefix)
    u = ref.half_step(dtype)
    u_p = ref.U16 if prefix is None else max(u, ref.U16)
    for b in range(B):
        for h in range(H):
            kk, vv = ref.values(c, b, h)
            scale = torch.exp2(c.scales[b, h, :, 1].double() - 127)
            if prefix is not None:
                kk, vv = torch.cat((prefix.k[h].double(), kk)), torch.cat((prefix.v[h].double(), vv))
            hs = slice(h * G, (h + 1) * G)
            eo, _, A, ds = ref.attention(q[b, hs, 0], kk, vv, LOG2)
            w = torch.softmax(q[b, hs, 0].double() @ kk.T * LOG2, -1)[:, -n:]
            extra = (w * scale).amax(-1)[:, None] * c.v[b, h].double().abs().sum(0) * 2.0 ** -36
            ref.check(o[b, hs, 0], eo, A, ds, u, u_p, extra, f"b{b} h{h}")


@pytest.mark.parametrize("H,n,G,ws", [(1, 40, 3, 0), (4, 6000, 2, 1)])
def test_scores_of_minus_infinity_only(H, n, G, ws):
    """A sequence whose every score overflows to minus infinity has tokens: it gives the NaN and the
    LSE of minus infinity that the formula gives, not an empty sequence's zeros, and behind a
    prefix what the prefix gives alone."""
    D, B, dt = 128, 36, torch.bfloat16
    c = Cache(B, H, D, 4, n - 4, dtype=dt, device=DEV)
    assert (native.lib().sbfa_qcache_attend_workspace_bytes(c._handle, H * G) > 0) == bool(ws)
    k, v = torch.zeros(B, H, n, D, dtype=dt, device=DEV), rows(gen(45), (B, H, n, D), dt)
    q = torch.zeros(B, H * G, 1, D, dtype=dt, device=DEV)
    q[..., 0], k[..., 0] = 3e38, -3e38
    counts = torch.full((B,), n, device=DEV)
    counts[::3] = 0
    counts[1::3] = torch.arange(1, n, n // 12, device=DEV)[:12]
    c.append(k, v, counts)
    o, lse = c.attend(q, return_lse=True)
    some = counts > 0
    assert not o[~some].any() and not lse[~some].any()
    assert torch.isnan(o[some]).all() and (lse[some] == -math.inf).all()
    pre = SharedPrefix(torch.zeros(H, 70, D, dtype=dt, device=DEV), rows(gen(46), (H, 70, D), dt))
    o, lse = c.attend(q, return_lse=True, prefix=pre)
    c.reset()
    alone = c.attend(q, return_lse=True, prefix=pre)
    assert torch.equal(o, alone[0]) and torch.equal(lse, alone[1])
