"""Plain 64-bit forms of the 8-bit ring cache and of attention to a shared prefix, written from
their definitions, and the error bounds the tests hold the kernels to.

Bounds.  With u = eps / 2 of the output type (half a step), A = sum_j w_j |v_j| (w: the softmax's
weights) and ds the error of a score, an output may differ from the exact one by
    u |o|                 the rounding of the output,
    A * u_p               the rounding of the weights to u_p (fp16 in the cache's kernel, the
                          input type in the prefix's), which are summed with |v|,
    2 A ds                wrong scores (each weight, and their sum),
    A * 2^-17             exponentials and sums in fp32: an argument below 2^7 is off by half of its
                          last place, 2^-18, and the approximate 2^x by 2^-22.
A score is a sum of D products in fp32: each addition is off by at most one last place (the
tensor core truncates), so ds = D 2^-23 sum |q_d k_d| scale.  Weights of fp16 below 2^-14 of the
largest are off by 2^-25 absolutely: n 2^-25 times the largest scaled value.
"""

from __future__ import annotations

import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
U16 = 2.0 ** -11   # half a step of fp16, relative


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantise(x: torch.Tensor, fmt: str):
    """Codes (as float64) and scale bytes of the rows of x, from the definition."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, -126)
    for _ in range(260):  # the least e that holds the row
        e = torch.where(amax > TOP[fmt] * torch.exp2(e), e + 1, e)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = x * torch.exp2(-e)[..., None]
    if fmt == "int8":
        codes = torch.round(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        codes = torch.round(y / step) * step
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return codes, byte.to(torch.uint8)


def ring_row(p: int, sink: int, window: int) -> int:
    return p if p < sink else sink + (p - sink) % window


def kept_positions(length: int, sink: int, window: int):
    return [p for p in range(length) if p < sink or p >= length - window]


def values(cache, b: int, h: int):
    """Float64 K and V of all ring rows of (b, h), NaN for bad rows."""
    out = []
    for part, codes in ((0, cache.k), (1, cache.v)):
        byte = cache.scales[b, h, :, part].double()
        x = codes[b, h].double() * torch.exp2(byte - 127)[:, None]
        out.append(torch.where((byte == 255)[:, None], torch.full_like(x, math.nan), x))
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """q [G, D] over keys [n, D] in float64: O, LSE (-inf where there is no key), the weighted
    mean of |v|, and the bound of a score's error."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        g = torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
        return z, g - math.inf, z, g
    x = q @ k.T * scale
    w = torch.softmax(x, -1)
    ds = (q.abs() @ k.abs().T).amax(-1) * scale * q.shape[-1] * 2.0 ** -23
    return w @ v, torch.logsumexp(x, -1), w @ v.abs(), ds


def check(o, ref, A, ds, u_out: float, u_p: float, extra: float = 0.0, label: str = ""):
    o, ref = o.double(), ref.double()
    assert torch.isfinite(o).all(), f"{label}: non-finite output"
    tol = u_out * ref.abs() + A * (u_p + 2 * ds[..., None] + 2.0 ** -17) + extra + 1e-30
    bad = ((o - ref).abs() / tol).max().item()
    assert bad <= 1.0, f"{label}: error is {bad:.3g} of its bound"


def check_lse(lse, ref, ds, label: str = ""):
    tol = ds + 2.0 ** -17 * (1 + ref.abs())
    bad = ((lse.double() - ref).abs() / tol).max().item()
    assert bad <= 1.0, f"{label}: LSE error is {bad:.3g} of its bound"
