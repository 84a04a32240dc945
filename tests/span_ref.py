"""Definitions in 64 bits of the 4-bit rows and of attention under a window with sinks, and the
bounds on what a kernel of 16- or 32-bit operands may be off by."""
from __future__ import annotations

import math

import torch

CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E_HIGH = {torch.float16: 13, torch.bfloat16: 125}


def pack_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(code values 0..15 [..., D], scale bytes [..., D/32]) of fp16 / bf16 rows on the CPU, by
    trying every code; non-finite blocks get code 0 and scale 255."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    e = torch.full(top.shape, E_HIGH[x.dtype], dtype=torch.long)
    for t in range(E_HIGH[x.dtype] - 1, -24, -1):
        e = torch.where(top <= 7.0 * 2.0 ** t, torch.full_like(e, t), e)
    a = (b.abs() / torch.pow(2.0, e.double())[..., None]).clamp(max=6.0)
    a = torch.where(finite[..., None], a, 0.0)
    dist = (a[..., None] - CODES).abs()
    # the nearest code; of two equally near the even one
    near = dist == dist.amin(-1, keepdim=True)
    rank = near.double() * torch.tensor([2.0, 1.0] * 4, dtype=torch.float64)
    code = rank.argmax(-1) + 8 * (torch.signbit(b) & finite[..., None]).long()
    return code.flatten(-2), torch.where(finite, e + 127, 255).to(torch.uint8)


def values_of(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    v = torch.where(code >= 8, -CODES[code % 8], CODES[code % 8]).unflatten(-1, (-1, 32))
    f = torch.where(scale == 255, torch.full(scale.shape, math.nan, dtype=torch.float64),
                    torch.pow(2.0, scale.double() - 127))
    return (v * f[..., None]).flatten(-2)


def round4(x: torch.Tensor) -> torch.Tensor:
    """float64 values that 16-bit rows have in 4 bits."""
    return values_of(*pack_rows(x))


def sees(pos: torch.Tensor, n: int, window: int, sinks: int) -> torch.Tensor:
    """[len(pos), n]: which keys queries at positions pos see."""
    key = torch.arange(n)
    s = key <= pos[:, None]
    if window:
        s &= (pos[:, None] - key < window) | (key < sinks)
    return s


def attend(q, k, v, pos, window, sinks, scale=None):
    """float64 attention of q [m, Hq, D] at positions pos over k, v [n, Hkv, D], and its bound:
    elementwise |error| <= bound for the element type of q."""
    m, hq, d = q.shape
    n, hkv, _ = k.shape
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    see = sees(pos, n, window, sinks)
    qd = q.double().reshape(m, hkv, g, d)
    kd, vd = k.double(), v.double()
    any_seen = see.any(0)[:, None, None]
    kd, vd = torch.where(any_seen, kd, 0.0), torch.where(any_seen, vd, 0.0)
    x = torch.einsum("mhgd,nhd->mhgn", qd, kd) * scale
    w = torch.softmax(x.masked_fill(~see[:, None, None], -math.inf), -1)
    out = torch.einsum("mhgn,nhd->mhgd", w, vd).reshape(m, hq, d)
    # A score's error from D products and sums in 32 bits; a probability's is that much relative
    # (both ways: numerator and sum), its rounding to 16 bits, and the exponential's; sums of n
    # terms pass through at most n / 16 + 64 additions in a row; fp16 probabilities below 2^-14
    # are off by up to 2^-25 each beside a largest of at least 1.
    mags = torch.einsum("mhgd,nhd->mhgn", qd.abs(), kd.abs()) * abs(scale)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[q.dtype]
    ds = (d + 4) * 2.0 ** -24 * mags.masked_fill(~see[:, None, None], 0).amax(-1)
    rel = 2 * ds + 2.0 ** -21 + (n / 16 + 64) * 2.0 ** -24
    if q.dtype != torch.float32:
        rel = rel + u
    if q.dtype == torch.float16:
        rel = rel + see.sum(1)[:, None, None] * 2.0 ** -25
    vmax = torch.where(see[:, :, None], vd.abs().amax(-1)[None], 0.0).amax(1)    # [m, Hkv]
    bound = (rel * vmax[:, :, None])[..., None].expand(m, hkv, g, d).reshape(m, hq, d)
    return out, bound + u * out.abs() + (2.0 ** -25 if q.dtype == torch.float16 else 1e-38)


def assert_close(got, out, bound, what=""):
    got = got.double().cpu()
    assert got.shape == out.shape, (got.shape, out.shape)
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    over = ((got - out).abs() - bound)
    worst = over.argmax()
    assert over.max() <= 0, (f"{what}: off by {(got - out).abs().flatten()[worst]:.3e} where "
                             f"{bound.flatten()[worst]:.3e} is allowed")
