"""Prompts behind a shared prefix: infinities that meet slices of a row's keys, padding, and sinks,
against 64 bits within the bounds of ``serving_reference``."""

from __future__ import annotations

import math

import pytest
import torch

import sbfa_native as native
from shared_prefix import SharedPrefix
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
