"""CPU: which layouts a 4-bit pool may have -- what Kv4Pool takes and refuses, and what the
_strided entry points refuse on the host."""
from __future__ import annotations

import ctypes

import pytest
import torch

from flexengine_amd import _lib, ops
from tests.test_span_host import INVALID, UNSUPPORTED, WORKSPACE, P, lib  # noqa: F401

NB, HKV, BS, D = 5, 2, 16, 128


def tensors(order, last=1, gap=0, nb=NB, hkv=HKV, bs=BS, d=D):
    """codes and scales [nb, hkv, bs, *] whose dims lie in memory in `order` (of b, h, t), the rows
    `gap` bytes (codes; of scales an eighth) apart; last: the stride within a row."""
    size = dict(b=nb, h=hkv, t=bs)
    out = []
    for n, g in ((d // 2, gap), (d // 32, gap // 8)):
        x = torch.zeros([size[c] for c in order] + [(n + g) * last], dtype=torch.uint8)
        out.append(x.permute([order.index(c) for c in "bht"] + [3])[..., :n * last:last])
    return out


def pool(order, **kw):
    return ops.Kv4Pool(*tensors(order, **kw), torch.float16)


@pytest.mark.parametrize("order", ["bht", "bth", "hbt", "tbh", "thb", "htb"])
@pytest.mark.parametrize("gap", [0, 16])
def test_any_order_of_the_dims_and_gaps_are_taken(order, gap):
    p = pool(order, gap=gap)
    assert p.layout() == (NB, BS, HKV, D) and p.shape == (NB, BS, HKV, D)
    assert ops._check_pool4(p, pool(order, gap=gap)) == (NB, BS, HKV, D)


def test_layers_of_any_layout_are_pools_of_their_own():
    codes, scales = tensors("bth")
    many = ops.Kv4Pool(torch.stack((codes, codes)).transpose(0, 1).contiguous().transpose(0, 1),
                       torch.stack((scales, scales)), torch.float16)
    assert many[1].layout() == (NB, BS, HKV, D) and many[1].codes.stride(0) == 2 * HKV * BS * D // 2


def test_layouts_of_what_prepares_rows_by_token_are_taken():
    # rows [blocks, tokens, heads, dims] packed through a transposed view, as elementwise
    # operations leave them: codes by token, and scales in either order
    for hkv, d, bs in ((2, 128, 16), (8, 64, 16), (4, 96, 32), (1, 32, 16)):
        x = torch.randn(3, bs, hkv, d).transpose(1, 2)
        codes = (x[..., 0::2] > 0).to(torch.uint8) | (x[..., 1::2] > 0).to(torch.uint8) << 4
        scales = x.unflatten(-1, (-1, 32)).abs().amax(-1).to(torch.uint8)
        assert ops.Kv4Pool(codes, scales).layout() == (3, bs, hkv, d)


def test_refused_layouts():
    for bad in (dict(last=2), dict(gap=8)):       # bytes of a row apart; rows at odd places
        with pytest.raises(ValueError):
            pool("bht", **bad).layout()
    codes, scales = tensors("bht")
    for c, s in ((codes[:, :1].expand(NB, HKV, BS, D // 2), scales),     # heads share their rows
                 (codes, scales[:1].expand(NB, HKV, BS, D // 32)),
                 (codes.as_strided(codes.shape, (HKV * BS * 64, BS * 64, 32, 1)), scales)):
        with pytest.raises(ValueError):
            ops.Kv4Pool(c, s, torch.float16).layout()
    with pytest.raises(ValueError):               # K in one layout, V in another
        ops._check_pool4(pool("bht"), pool("bth"))


class Strides(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_int64 * 3), ("scales", ctypes.c_int64 * 3)]


def strides(c=(4096, 64, 128), s=(256, 4, 8)):
    return ctypes.cast(ctypes.pointer(Strides(c, s)), ctypes.c_void_p)


BAD = [dict(c=(4096, 32, 128)), dict(c=(4096, 64, 64)), dict(c=(2032, 64, 128)), dict(c=(4096, 72, 144)),
       dict(c=(-4096, 64, 128)), dict(s=(256, 0, 8)), dict(s=(127, 4, 8)), dict(s=(256, 4, -8)),
       dict(c=(1 << 62, 1 << 62, 1 << 62))]
FAR = [dict(c=(1 << 36, 64, 128)), dict(s=(1 << 32, 4, 8)), dict(c=(64, 1024, 1 << 26)),
       dict(s=(4, 64, 1 << 26))]


@pytest.mark.parametrize("sfx", ["", "_bf16"])
def test_strided_forms_refuse_on_the_host(lib, sfx):  # noqa: F811
    pools = (P, P, P, P)

    def write(st, n=3):
        return getattr(lib, "fe_write_kv4_strided" + sfx)(P, P, 256, *pools, st, 9, P, P, n, 2, 128, 16, None)

    def dec(st, n=3):
        return getattr(lib, "fe_write_kv4_decode_strided" + sfx)(P, P, 256, *pools, st, 9, P, 4, P, n, 2, 128,
                                                                 16, None)

    def rag(st, n=3):
        return getattr(lib, "fe_write_kv4_ragged_strided" + sfx)(P, P, 256, *pools, st, 9, P, 4, P, P, 2, n, 2,
                                                                 128, 16, None)

    def gather(st, n=3):
        return getattr(lib, "fe_gather_kv4_strided" + sfx)(*pools, st, 9, P, 4, P, P, P, P, 2, n, 2, 128, 16, None)

    def decode(st, n=2):
        return getattr(lib, "fe_paged_decode_kv4_strided" + sfx)(
            P, 1536, P, None, None, 0, *pools, st, 9, P, 4, P, P, 0, n, 12, 2, 128, 16, 0.1, 8, 0, 0, None)

    def prefill(st, n=9):
        return getattr(lib, "fe_prefill_paged_kv4_strided" + sfx)(
            P, P, *pools, st, 9, P, 4, P, P, 2, n, 12, 2, 128, 16, 0.1, 8, 0, P, 0, None)

    for f in (write, dec, rag, gather, decode, prefill):
        for bad in BAD:
            assert f(strides(**bad)) == INVALID, (f, bad)
        for far in FAR:
            assert f(strides(**far)) == UNSUPPORTED, (f, far)
        assert f(strides(), n=0) == _lib.FE_OK
    for f in (decode, prefill):   # past the strides: what the dense forms come to
        assert f(strides()) == WORKSPACE and f(None) == WORKSPACE
