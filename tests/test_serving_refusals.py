"""Refusals of the 8-bit ring cache and the shared prefix that need no GPU: the C entry points'
argument checks (nothing is launched) and the Python classes' own."""

from __future__ import annotations

import ctypes

import pytest
import torch

import sbfa_native as native

INVALID, UNSUPPORTED = 1, 2
P = 4096   # a non-null, 16-byte aligned address that is never read


def cache(B=1, H=1, D=64, dtype=native.BF16, fmt=0, sink=4, window=8, k=P, tickets=P):
    c = native.QCache(k, P, P, P, tickets, B, H, D, sink, window, dtype, fmt)
    return c, ctypes.addressof(c)


def append(L, n=1, new=P, strides=None, **kw):
    st = None if strides is None else (ctypes.c_int64 * 6)(*strides)
    keep, at = cache(**kw)
    return L.sbfa_qcache_append(at, new, P, st, None, n, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(dtype=native.F32), UNSUPPORTED, "float16"), (dict(fmt=2), INVALID, "format"),
    (dict(B=0), INVALID, "positive"), (dict(H=0), INVALID, "positive"),
    (dict(B=65536), UNSUPPORTED, "65535"), (dict(H=1 << 60), UNSUPPORTED, "heads"),
    (dict(sink=1 << 62, window=1 << 62), INVALID, "2^30"), (dict(D=0), UNSUPPORTED, "head_dim"),
    (dict(D=60), UNSUPPORTED, "head_dim"), (dict(D=264), UNSUPPORTED, "head_dim"),
    (dict(sink=-1), INVALID, "non-negative"), (dict(sink=0, window=0), INVALID, "2^30"),
    (dict(window=1 << 30), INVALID, "2^30"), (dict(k=None), INVALID, "NULL"),
    (dict(k=P + 8), INVALID, "aligned"), (dict(n=-1), INVALID, "n_new"),
    (dict(new=None), INVALID, "NULL"), (dict(new=P + 2), INVALID, "aligned"),
    (dict(tickets=None), INVALID, "NULL"),
    (dict(strides=(64, 64, 60, 64, 64, 64)), INVALID, "strides"),
    (dict(strides=(64, 64, 64, -64, 64, 64)), INVALID, "strides"),
])
def test_append_refuses(kw, rc, word):
    assert append(native.lib(), **kw) == rc and word in native.last_error()


def test_append_of_nothing_launches_nothing():
    before = native.launch_count()
    assert append(native.lib(), n=0, new=None) == 0 and native.launch_count() == before


def test_a_null_cache_is_refused():
    L = native.lib()
    assert L.sbfa_qcache_append(None, P, P, None, None, 1, None) == INVALID
    assert L.sbfa_qcache_attend(None, P, P, None, 4, 0.1, None, 0, None) == INVALID
    assert L.sbfa_qcache_read(None, P, P, P, None) == INVALID
    assert L.sbfa_qcache_prefix_attend(None, P, P, P, 9, P, None, 4, 0.1, P, 99, None) == INVALID
    assert L.sbfa_qcache_attend_workspace_bytes(None, 4) == -1
    assert L.sbfa_qcache_prefix_workspace_bytes(None, 4, 9) == -1


def attend(L, q=P, o=P, lse=P, B=1, H=4, hkv=2, scale=0.1, ws=P, ws_bytes=1 << 40, window=8):
    keep, at = cache(B=B, H=hkv, window=window, dtype=native.F16, fmt=1)
    return L.sbfa_qcache_attend(at, q, o, lse, H, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,word", [
    (dict(H=3), "multiple"), (dict(H=0), "multiple"), (dict(scale=0.0), "softmax_scale"),
    (dict(scale=-1.0), "softmax_scale"), (dict(scale=float("nan")), "softmax_scale"),
    (dict(scale=float("inf")), "softmax_scale"), (dict(q=None), "NULL"), (dict(o=None), "NULL"),
    (dict(q=P + 8), "aligned"),
    (dict(o=P + 4), "aligned"), (dict(B=300, window=9999, ws=None), "workspace"),
    (dict(B=300, window=9999, ws_bytes=1000), "workspace"), (dict(ws=P + 8), "aligned"),
])
def test_attend_refuses(kw, word):
    assert attend(native.lib(), **kw) == INVALID and word in native.last_error()


def prefix(L, q=P, k=P, own=None, own_lse=None, B=2, H=4, hkv=2, n=1, length=100, D=64,
           dtype=native.F16, scale=0.1, ws=P, ws_bytes=1 << 40, strides=None):
    st = None if strides is None else (ctypes.c_int64 * 3)(*strides)
    return L.sbfa_prefix_attend(q, st, k, P, own, own_lse, P, P, B, H, hkv, n, length, D,
                                dtype, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(dtype=native.F32), UNSUPPORTED, "float16"), (dict(D=136), UNSUPPORTED, "head_dim"),
    (dict(D=12), UNSUPPORTED, "head_dim"), (dict(H=3), INVALID, "multiple"),
    (dict(length=0), INVALID, "positive"), (dict(n=0), INVALID, "positive"),
    (dict(length=1 << 31), INVALID, "positive"), (dict(scale=0.0), INVALID, "softmax_scale"),
    (dict(q=None), INVALID, "NULL"), (dict(own=P), INVALID, "own"),
    (dict(own_lse=P), INVALID, "own"),
    (dict(k=P + 8), INVALID, "aligned"), (dict(ws=None, length=9000), INVALID, "workspace"),
    (dict(ws_bytes=16, length=9000), INVALID, "workspace"), (dict(strides=(64, 64, 4)), INVALID, "strides"),
    (dict(strides=(64, -8, 8)), INVALID, "strides"),
])
def test_prefix_refuses(kw, rc, word):
    assert prefix(native.lib(), **kw) == rc and word in native.last_error()


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=136), UNSUPPORTED, "head_dim"), (dict(dtype=native.F32), UNSUPPORTED, "float16"),
    (dict(fmt=7), INVALID, "format"), (dict(H=3), INVALID, "multiple"),
    (dict(length=0), INVALID, "positive"), (dict(ws=None), INVALID, "workspace"),
    (dict(ws_bytes=256), INVALID, "workspace"), (dict(k=None), INVALID, "NULL"),
    (dict(q=P + 8), INVALID, "aligned"), (dict(scale=0.0), INVALID, "softmax_scale"),
])
def test_decode_behind_a_prefix_refuses(kw, rc, word):
    a = dict(q=P, k=P, H=4, length=100, D=64, dtype=native.F16, fmt=0, scale=0.1, ws=P,
             ws_bytes=1 << 40) | kw
    keep, at = cache(B=2, H=2, D=a["D"], dtype=a["dtype"], fmt=a["fmt"])
    got = native.lib().sbfa_qcache_prefix_attend(at, a["q"], a["k"], P, a["length"], P, None,
                                                 a["H"], a["scale"], a["ws"], a["ws_bytes"], None)
    assert got == rc and word in native.last_error()


def test_sizes():
    L = native.lib()
    assert [L.sbfa_qcache_row_bytes(d) for d in (0, 8, 64, 72, 128, 136, 256, 264, 60)] == \
        [0, 64, 64, 128, 128, 256, 256, 0, 0]
    # one key tile is never cut; a long prefix before few rows is
    assert L.sbfa_prefix_workspace_bytes(2, 4, 2, 1, 100, 64, 0) == 0
    assert L.sbfa_prefix_workspace_bytes(2, 4, 2, 1, 9000, 64, 0) >= 2 * 2 * 256 * (64 * 4 + 8)
    for bad in ((0, 4, 2, 1, 100, 64, 0), (2, 4, 3, 1, 100, 64, 0), (2, 4, 2, 1, 0, 64, 0),
                (2, 4, 2, 1, 100, 256, 0), (2, 4, 2, 1, 100, 64, -1)):
        assert L.sbfa_prefix_workspace_bytes(*bad) == -1

    def bytes_of(H=4, P=None, **kw):
        keep, at = cache(**({"B": 2, "H": 2} | kw))
        return (L.sbfa_qcache_attend_workspace_bytes(at, H) if P is None
                else L.sbfa_qcache_prefix_workspace_bytes(at, H, P))

    assert bytes_of(P=100) >= 2 * 4 * 65 * 4
    assert bytes_of(H=3, P=100) == -1 and bytes_of(D=136, P=100) == -1
    # few units share clusters and need no scratch, many long ones are cut into equal runs
    assert bytes_of() == 0 and bytes_of(B=300, window=9999) > 0
    for bad in (dict(H=3), dict(D=60), dict(B=0), dict(sink=0, window=0), dict(sink=1 << 62),
                dict(B=1 << 40)):
        kw = {k: v for k, v in bad.items() if k != "H"}
        assert bytes_of(H=bad.get("H", 4), **kw) == -1


@pytest.mark.parametrize("kw,word", [
    (dict(window=0), "window"), (dict(k=None), "NULL"), (dict(k=P + 8), "k and v"),
    (dict(strides=(64,) * 3 + (64, 0, 64) + (64,) * 3), "k and v"),
    (dict(strides=(64,) * 3 + (64,) * 3 + (64, 64, 12)), "k and v"),
    (dict(strides=(64, 64, -8) + (64,) * 6), "strides"), (dict(n=0), "positive"),
    (dict(length=9000, ws=None), "workspace"),
])
def test_prompt_refuses(kw, word):
    a = dict(k=P, window=4, strides=None, n=3, length=100, ws=P) | kw
    st = None if a["strides"] is None else (ctypes.c_int64 * 9)(*a["strides"])
    rc = native.lib().sbfa_prefix_prompt(P, a["k"], P, st, P, P, P, None, 2, 4, 2, a["n"],
                                         a["length"], 64, native.BF16, 0.1, a["window"], a["ws"],
                                         1 << 40, None)
    assert rc == INVALID and word in native.last_error()


def test_python_refusals():
    from shared_prefix import SharedPrefix
    from streaming_kv_cache import QuantizedStreamingKVCache as Cache
    for args, kw in (((0, 1, 64, 4, 8), {}), ((1, 1, 64, -1, 8), {}), ((1, 1, 64, 0, 0), {}),
                     ((1, 1, 60, 4, 8), {}), ((1, 1, 512, 4, 8), {}),
                     ((1, 1, 64, 4, 8), dict(dtype=torch.float32)),
                     ((1, 1, 64, 4, 8), dict(fmt="e5m2")),
                     ((1, 1, 64, 4, 8), dict(device="cpu"))):
        with pytest.raises(ValueError):
            Cache(*args, **kw)
    k = torch.zeros(2, 10, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        SharedPrefix(k, k)
    with pytest.raises(ValueError, match="empty"):
        SharedPrefix(k[:, :0], k[:, :0])
    with pytest.raises(ValueError, match="H_kv"):
        SharedPrefix(k[0], k[0])
