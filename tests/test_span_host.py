"""CPU: what the windowed and 4-bit entry points refuse on the host, the 4-bit cache's
bookkeeping, the definitions' own properties, and the ticket protocol of the new kernels."""
from __future__ import annotations

import ctypes
import math
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

from flexengine_amd import _lib, ops
from flexengine_amd import build as B
from flexengine_amd.kv_cache import CacheExhausted, CacheLayout, PagedKVCache
from tests import span_ref as R
from tests import test_isa_protocol as isa

P = ctypes.c_void_p(256)  # never dereferenced: validation fails first
INVALID, UNSUPPORTED, WORKSPACE = (_lib.FE_ERR_INVALID_ARGUMENT, _lib.FE_ERR_UNSUPPORTED,
                                   _lib.FE_ERR_WORKSPACE)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        B.build()
    return _lib.load()


def decode(lib, kind, sfx="", q=P, q_stride=1536, out=P, kn=None, vn=None, new_stride=0, pool=P,
           scales=P, nb=9, tables=P, width=4, ctx=P, ws=P, ws_bytes=0, batch=2, hq=12, hkv=2, d=128,
           bs=16, scale=0.1, window=8, sinks=0, splits=0):
    pools = (pool, scales, pool, scales) if kind == "kv4" else (pool, pool)
    return getattr(lib, f"fe_paged_decode_{kind}{sfx}")(
        q, q_stride, out, kn, vn, new_stride, *pools, nb, tables, width, ctx, ws, ws_bytes, batch, hq,
        hkv, d, bs, scale, window, sinks, splits, None)


def prefill(lib, kind, sfx="", q=P, out=P, pool=P, scales=P, nb=9, tables=P, width=4, offs=P, ctx=P,
            seqs=2, total=9, hq=12, hkv=2, d=128, bs=16, scale=0.1, window=8, sinks=0, ws=P, ws_bytes=0):
    pools = (pool, scales, pool, scales) if kind == "kv4" else (pool, pool)
    return getattr(lib, f"fe_prefill_paged_{kind}{sfx}")(
        q, out, *pools, nb, tables, width, offs, ctx, seqs, total, hq, hkv, d, bs, scale, window, sinks,
        ws, ws_bytes, None)


FORMS = [("window", ""), ("window", "_bf16"), ("window", "_f32"), ("kv4", ""), ("kv4", "_bf16")]


@pytest.mark.parametrize("kind,sfx", FORMS)
@pytest.mark.parametrize("call", [decode, prefill])
def test_attention_forms_refuse_on_the_host(lib, call, kind, sfx):
    go = lambda **kw: call(lib, kind, sfx, **kw)  # noqa: E731
    for bad in (dict(window=-1), dict(sinks=-1), dict(hq=13), dict(hkv=0), dict(d=0), dict(nb=0),
                dict(width=0), dict(pool=None), dict(tables=None), dict(ctx=None), dict(q=None),
                dict(out=None), dict(q=ctypes.c_void_p(264)), dict(pool=ctypes.c_void_p(264))):
        assert go(**bad) == INVALID, bad
    if kind == "window":
        assert go(window=0) == INVALID
    else:
        assert go(scales=None) == INVALID
    assert go(d=36) == UNSUPPORTED and go(d=512) == UNSUPPORTED
    assert go(d=48 if kind == "kv4" else 44) == UNSUPPORTED
    if sfx == "_f32":
        assert go(d=136) == UNSUPPORTED
    for bs in (8, 24, 0):
        assert go(bs=bs) == UNSUPPORTED, bs
    assert go(nb=1 << 30) == UNSUPPORTED               # pool rows past 32 bits
    assert go() == WORKSPACE and go(ws=None, ws_bytes=1 << 40) == WORKSPACE
    assert go(ws=ctypes.c_void_p(260), ws_bytes=1 << 40) == WORKSPACE


@pytest.mark.parametrize("kind,sfx", FORMS)
def test_decode_refuses_strides_new_rows_and_large_batches(lib, kind, sfx):
    go = lambda **kw: decode(lib, kind, sfx, **kw)  # noqa: E731
    assert go(q_stride=1528) == INVALID                # shorter than a row
    assert go(q_stride=1538) == INVALID                # not 16-byte rows
    assert go(kn=P) == INVALID and go(vn=P, new_stride=256) == INVALID
    assert go(kn=P, vn=P, new_stride=128) == INVALID
    assert go(kn=ctypes.c_void_p(258), vn=P, new_stride=256) == INVALID
    assert go(splits=-1) == INVALID
    assert go(width=32768) == UNSUPPORTED              # 524288 tokens
    assert go(batch=40000) == UNSUPPORTED              # more tickets than the workspace has
    assert go(batch=0) == _lib.FE_OK


@pytest.mark.parametrize("kind,sfx", FORMS)
def test_prefill_refuses_scales_and_takes_empty_steps(lib, kind, sfx):
    go = lambda **kw: prefill(lib, kind, sfx, **kw)  # noqa: E731
    for scale in (0.0, -1.0, math.nan):
        assert go(scale=scale) == INVALID
    assert go(total=-1) == INVALID and go(seqs=-1) == INVALID and go(offs=None) == INVALID
    assert go(width=1 << 27) == UNSUPPORTED
    assert go(total=0) == _lib.FE_OK and go(seqs=0) == _lib.FE_OK


@pytest.mark.parametrize("sfx", ["", "_bf16"])
def test_page_movers_refuse_on_the_host(lib, sfx):
    pools = (P, P, P, P)

    def write(k=P, stride=256, p=pools, nb=9, n=3, hkv=2, d=128, bs=16):
        return getattr(lib, "fe_write_kv4" + sfx)(k, P, stride, *p, nb, P, P, n, hkv, d, bs, None)

    def rag(k=P, stride=256, p=pools, nb=9, w=4, n=3, hkv=2, d=128, bs=16, s=2):
        return getattr(lib, "fe_write_kv4_ragged" + sfx)(k, P, stride, *p, nb, P, w, P, P, s, n, hkv, d,
                                                         bs, None)

    def dec(k=P, stride=256, p=pools, nb=9, w=4, n=3, hkv=2, d=128, bs=16):
        return getattr(lib, "fe_write_kv4_decode" + sfx)(k, P, stride, *p, nb, P, w, P, n, hkv, d, bs, None)

    def gather(k=P, p=pools, nb=9, w=4, n=3, hkv=2, d=128, bs=16):
        return getattr(lib, "fe_gather_kv4" + sfx)(*p, nb, P, w, P, P, k, P, 2, n, hkv, d, bs, None)

    for f in (write, rag, dec, gather):
        assert f(d=48) == UNSUPPORTED and f(bs=24) == UNSUPPORTED
        for bad in (dict(n=-1), dict(nb=0), dict(hkv=0), dict(d=0), dict(k=None),
                    dict(k=ctypes.c_void_p(264)), dict(p=(P, None, P, P)),
                    dict(p=(ctypes.c_void_p(264), P, P, P))):
            assert f(**bad) == INVALID, (f, bad)
        assert f(n=0) == _lib.FE_OK
    for f in (write, rag, dec):
        assert f(stride=255) == INVALID and f(stride=128) == INVALID
    for f in (rag, dec, gather):
        assert f(w=0) == INVALID
    assert rag(s=0) == _lib.FE_OK


def test_workspace_sizes(lib):
    size = lib.fe_span_decode_workspace_size
    assert size(-1, 12, 2, 128, 64, 0) == 0 and size(1, 12, 5, 128, 64, 0) == 0
    assert 0 < size(8, 12, 2, 128, 4096, 0) <= size(64, 12, 2, 128, 4096, 0)
    assert size(4, 12, 2, 96, 4096, 0) == size(4, 12, 2, 128, 4096, 0)   # computed as 128 dims
    size = lib.fe_span_prefill_workspace_size
    assert size(1, 10, 12, 5, 128) == 0 and size(1, 10, 12, 2, 128) > 0
    # key splits' rows stay bounded: a step with many rows has none
    assert size(4, 100000, 32, 8, 128) == 65536 * 4


def test_a_4_bit_cache_keeps_the_books_anywhere():
    cache = PagedKVCache(CacheLayout(2, 8, 16, 2, 64), device="cpu", bits=4)
    cache.reserve("a", 40)
    assert cache.k[1].shape == (8, 16, 2, 64) and cache.k[0].codes.shape == (8, 2, 16, 32)
    assert cache.k[0].scales.shape == (8, 2, 16, 2) and cache.v.shape == (2, 8, 16, 2, 64)
    assert cache.k[0].codes.data_ptr() == cache.k.codes.data_ptr()
    with pytest.raises(CacheExhausted):
        cache.reserve("b", 16 * 6)
    cache.assert_invariants()
    with pytest.raises(ValueError):
        PagedKVCache(CacheLayout(1, 4, 16, 2, 64), device="cpu", bits=8)
    with pytest.raises(ValueError):
        PagedKVCache(CacheLayout(1, 4, 16, 2, 64), device="cpu", bits=4, fill=float("nan"))
    with pytest.raises(ValueError):
        PagedKVCache(CacheLayout(1, 4, 16, 2, 48), device="cpu", bits=4)
    with pytest.raises(ValueError):
        PagedKVCache(CacheLayout(1, 4, 16, 2, 64), device="cpu", dtype=torch.float32, bits=4)
    with pytest.raises(RuntimeError):   # no kernels on the CPU
        cache.write(0, "a", 0, torch.zeros(1, 2, 64).half(), torch.zeros(1, 2, 64).half())


def test_window_arguments():
    assert ops.check_window(None) == (0, 0) and ops.check_window(5, 2) == (5, 2)
    assert ops.check_window(1 << 40, 1 << 40) == (1 << 30, 1 << 30)
    for bad in ((0, 0), (-1, 0), (4, -1), (None, 1)):
        with pytest.raises(ValueError):
            ops.check_window(*bad)
    with pytest.raises(TypeError):
        ops.check_window(2.5)


def test_the_4_bit_definition_rounds_to_the_nearest_value_held():
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).half()
    code, scale = R.pack_rows(x)
    v = R.values_of(code, scale)
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    e = torch.pow(2.0, scale.double() - 127)
    assert (top <= 7 * e).all() and (top > 3.5 * e).all()
    # every value is the nearest one that its block's scale can hold
    grid = torch.cat((R.CODES, -R.CODES)) * e[..., None, None]
    b = x.double().unflatten(-1, (-1, 32))[..., None]
    best = (grid - b).abs().amin(-1)
    assert torch.equal((v.unflatten(-1, (-1, 32)) - b[..., 0]).abs(), best)
    assert torch.equal(R.round4(v.half()), v) and torch.equal(v.half().double(), v)


def test_ticket_protocol_of_the_new_kernels():
    """The rules of tests/test_isa_protocol.py for the kernels that join splits."""
    files = {"span_decode.hip": ("span_decode_kernel",), "span_prefill.hip": ("span_prefill_kernel",),
             "kv4_prefill.hip": ("span_prefill_kernel",)}
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(max_workers=3) as pool:
        asms = pool.map(lambda f: isa._assemble(B.CSRC_DIR / f, Path(tmp) / (f + ".s"), B.CSRC_DIR), files)
        for (name, families), asm in zip(files.items(), asms):
            found, bad = isa.violations(asm)
            for family in families:
                assert any(family in k for k in found), f"{family} has no ticket in {name}"
            assert not bad, "\n".join(f"{n}: {r}" for n, r in bad)


def test_the_prefill_workspace_stays_small_for_many_sequences(lib):
    tickets = 65536 * 4
    for seqs, total, hq, hkv, d in ((4, 1500, 12, 2, 128), (1000, 1000, 12, 2, 128), (64, 1280, 32, 8, 256),
                                    (1, 1, 96, 96, 8), (1, 100000, 32, 8, 128), (5000, 5000, 8, 8, 64)):
        need = lib.fe_span_prefill_workspace_size(seqs, total, hq, hkv, d)
        assert tickets <= need <= tickets + (1 << 28), (seqs, total, need)
    assert lib.fe_span_prefill_workspace_size(1, 100000, 32, 8, 128) == tickets   # fills the chip unsplit
    assert lib.fe_span_prefill_workspace_size(4, 1500, 12, 2, 128) > tickets
