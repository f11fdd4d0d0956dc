"""Refusals of the prompt entry point with own sinks, which launch nothing and need no GPU."""

from __future__ import annotations

import pytest

import sbfa_native as native

P = 4096   # a non-null, 16-byte aligned address that is never read


def prompt(k=P, n=3, length=100, sink=4, window=4, ws=P):
    return native.lib().sbfa_prefix_prompt_sinks(P, k, P, None, P, P, P, None, 2, 4, 2, n, length, 64,
                                                 native.BF16, 0.1, sink, window, ws, 1 << 40, None)


@pytest.mark.parametrize("kw,word", [
    (dict(sink=-1), "sink"), (dict(window=0), "window"), (dict(k=None), "NULL"),
    (dict(k=P + 8), "k and v"), (dict(n=0), "positive"), (dict(length=9000, ws=None), "workspace"),
    (dict(sink=1 << 40, window=0), "window"),
])
def test_prompt_with_sinks_refuses(kw, word):
    before = native.launch_count()
    assert prompt(**kw) == 1 and word in native.last_error()
    assert native.launch_count() == before
