"""GPU: windows with sinks and 4-bit caches through the package's own paths -- the cache, the
attention-backend calls, the Qwen2 forwards and the captured decode step -- against a dense
float64 forward that attends the rows the cache holds."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from flexengine_amd import attention, ops
from flexengine_amd.decode_step import GraphDecodeStep
from flexengine_amd.kv_cache import CacheLayout, PagedKVCache
from flexengine_amd.model import Chunk, Qwen2Config, Qwen2Model
from oracle.qwen2_ref import rotate_half
from tests import span_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# fp16 activations through every layer against float64: as the plain model's tests
MAX_REL, MEAN_REL = 5e-3, 1e-3


def tiny(window, sinks, d=64, hq=4, hkv=2, layers=2):
    cfg = Qwen2Config(vocab_size=320, hidden_size=hq * d, intermediate_size=192,
                      num_hidden_layers=layers, num_attention_heads=hq, num_key_value_heads=hkv,
                      head_dim=d, sliding_window=window, attention_sinks=sinks)
    return Qwen2Model(cfg, DEV, seed=7, std=0.1)


def cache_for(model, bits, blocks=64, bs=16):
    layout = CacheLayout(model.layers, blocks, bs, model.nkv, model.dim)
    return PagedKVCache(layout, device=DEV, bits=bits, fill=None if bits else float("nan"))


def dense_logits(model, ids, cache, rid):
    """Last-token logits (float64, CPU) of `ids`.  With a 4-bit cache the attention takes the
    K/V rows that the cache holds of `rid`, after checking each against this forward's own row:
    within half the distance between codes (at most max / 3.5 of its block of 32) and the fp16
    forward's error."""
    cfg, nq, nkv, dim, f64 = model.cfg, model.nq, model.nkv, model.dim, torch.float64
    w = lambda t: t.detach().to("cpu", f64)  # noqa: E731
    n = len(ids)
    x = w(model.embed)[torch.tensor(ids)]
    inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, dim, 2, dtype=f64) / dim))
    ang = torch.outer(torch.arange(n, dtype=f64), inv)
    cos, sin = torch.cat((ang, ang), -1).cos()[:, None], torch.cat((ang, ang), -1).sin()[:, None]
    norm = lambda t, g: w(g) * (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps))  # noqa: E731
    see = R.sees(torch.arange(n), n, cfg.sliding_window or 0, cfg.attention_sinks)
    for layer, lw in enumerate(model.layer_weights):
        qkv = norm(x, lw.input_norm) @ w(lw.w_qkv).t() + w(lw.b_qkv)
        q = qkv[:, :nq * dim].reshape(n, nq, dim)
        k = qkv[:, nq * dim:(nq + nkv) * dim].reshape(n, nkv, dim)
        v = qkv[:, (nq + nkv) * dim:].reshape(n, nkv, dim)
        q, k = q * cos + rotate_half(q) * sin, k * cos + rotate_half(k) * sin
        if cache.bits == 4:
            held = [w(t) for t in cache.materialize(layer, rid, n)]
            for t, h in zip((k, v), held):
                top = t.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
                off = (t - h).unflatten(-1, (-1, 32)).abs()
                assert (off <= top / 3.5 + 2e-2 * t.abs().max()).all()
            k, v = held
        o = torch.empty(n, nq, dim, dtype=f64)
        for h in range(nq):
            s = (q[:, h] @ k[:, h // (nq // nkv)].T) / math.sqrt(dim)
            o[:, h] = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ v[:, h // (nq // nkv)]
        x = x + o.reshape(n, nq * dim) @ w(lw.w_o).t()
        gu = norm(x, lw.post_norm) @ w(lw.w_gate_up).t()
        x = x + (F.silu(gu[:, :cfg.intermediate_size]) * gu[:, cfg.intermediate_size:]) @ w(lw.w_down).t()
    return (norm(x[-1:], model.final_norm) @ w(model.lm_head).t())[0]


def close(got, want):
    scale = want.abs().max().item()
    err = (got.double().cpu() - want).abs()
    assert err.max().item() <= MAX_REL * scale and err.mean().item() <= MEAN_REL * scale


SETUPS = [(None, 0, 4), (24, 3, 4), (24, 3, None), (7, 0, None)]


def tokens(n, seed):
    return torch.randint(0, 320, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("window,sinks,bits", SETUPS)
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 6, 1)])
def test_forward_whole_in_chunks_and_together(window, sinks, bits, d, hq, hkv):
    model = tiny(window, sinks, d, hq, hkv)
    cache = cache_for(model, bits)
    a, b = tokens(75, 1), tokens(9, 2)
    cache.reserve("a", 75), cache.reserve("b", 9)
    got = model.forward([Chunk("a", a, 0), Chunk("b", b, 0)], cache)
    close(got[0], dense_logits(model, a, cache, "a"))
    close(got[1], dense_logits(model, b, cache, "b"))
    cache.free_request("a")
    cache.reserve("a", 75)
    model.forward([Chunk("a", a[:31], 0)], cache)
    model.forward([Chunk("a", a[31:74], 31)], cache)
    last = model.forward([Chunk("b", tokens(1, 3), 8), Chunk("a", a[74:], 74)], cache)[1]
    close(last, dense_logits(model, a, cache, "a"))
    cache.assert_invariants()


@pytest.mark.parametrize("window,sinks,bits", SETUPS)
def test_captured_decode_steps_equal_eager_ones_and_the_dense_forward(window, sinks, bits):
    model = tiny(window, sinks)
    cache, other = cache_for(model, bits), cache_for(model, bits)
    seqs = [tokens(n, 10 + n) for n in (40, 5, 61)]
    for c in (cache, other):
        for i, ids in enumerate(seqs):
            c.reserve(f"r{i}", len(ids) + 8)
            model.forward([Chunk(f"r{i}", ids, 0)], c)
    step = GraphDecodeStep(model, cache, max_model_len=128)
    for t in range(6):
        new = tokens(3, 50 + t)
        chunks = [Chunk(f"r{i}", [new[i]], len(seqs[i])) for i in range(3)]
        out = step(chunks)                    # the bucket of four rows, one of them padding
        assert out is not None
        # the same step eagerly on the other cache, padded the same way
        tables = other.device_tables([f"r{i}" for i in range(3)] + [None], 8, pad_block=0)
        eager = model.decode_static(torch.tensor(new + [0], device=DEV),
                                    torch.tensor([len(s) for s in seqs] + [0], device=DEV), tables,
                                    torch.tensor([1., 1., 1., 0.], device=DEV), other)
        for i in range(3):
            seqs[i].append(new[i])
            assert torch.equal(out[i], eager[i])
        assert torch.count_nonzero(eager[3]) == 0
    assert step.manager.stats()["captures"] == 1 and step.manager.stats()["replays"] == 6
    for i in range(3):
        close(out[i], dense_logits(model, seqs[i], cache, f"r{i}"))


@pytest.mark.parametrize("bits", [4, None])
def test_backend_calls_agree_with_the_definition(bits):
    layout = CacheLayout(2, 40, 16, 2, 128)
    cache = PagedKVCache(layout, device=DEV, dtype=torch.bfloat16, bits=bits)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(90, 2, 128, generator=g).bfloat16() for _ in range(2))
    cache.reserve("x", 90)
    cache.tables["x"] = list(reversed(cache.tables["x"]))
    cache.write(1, "x", 0, k[:50].to(DEV), v[:50].to(DEV))
    cache.write(1, "x", 50, k[50:].to(DEV), v[50:].to(DEV))
    kd, vd = (R.round4(k), R.round4(v)) if bits else (k.double(), v.double())
    for got, want in zip(cache.materialize(1, "x", 90), (kd, vd)):
        assert torch.equal(got.double().cpu(), want)
    q = torch.randn(11, 12, 128, generator=g).bfloat16()
    pos = torch.arange(79, 90)
    for window, sinks in ((None, 0), (20, 3)):
        kw = dict(window=window, sinks=sinks)
        out, bound = R.attend(q, kd, vd, pos, window or 0, sinks)
        got = attention.attention_for_request(q.to(DEV), cache, 1, "x", 90, pos.to(DEV), **kw)
        R.assert_close(got, out, bound)
        one = attention.attention_for_request(q[-1:].to(DEV), cache, 1, "x", 90, pos[-1:].to(DEV), **kw)
        R.assert_close(one, out[-1:], bound[-1:])
        tables = cache.block_table(["x"]).long()
        batch = attention.paged_decode_batch(q[-1:].to(DEV), cache, 1, tables, pos[-1:].to(DEV),
                                             torch.ones(1, device=DEV), **kw)
        assert torch.equal(batch, one)
        offs = torch.tensor([0, 11], dtype=torch.int32, device=DEV)
        ctx = torch.tensor([90], dtype=torch.int32, device=DEV)
        ragged = attention.prefill_batch(q.to(DEV), cache, 1, tables.int(), offs, ctx, 11, **kw)
        R.assert_close(ragged, out, bound)


def test_a_4_bit_cache_shares_prefix_blocks_and_refuses_views():
    model = tiny(24, 3)
    cache = cache_for(model, 4)
    ids = tokens(40, 20)
    cache.reserve("a", 48)
    model.forward([Chunk("a", ids, 0)], cache)
    cache.attach_prefix("b", cache.tables["a"][:2])
    cache.reserve("b", 48)
    got = model.forward([Chunk("b", ids[32:], 32)], cache)[0]
    close(got, dense_logits(model, ids, cache, "b"))
    with pytest.raises(ValueError):
        list(cache.iter_blocks(0, "a", 16))
    with pytest.raises(RuntimeError):
        cache.write(0, "b", 0, torch.zeros(1, 2, 64, dtype=torch.float16, device=DEV),
                    torch.zeros(1, 2, 64, dtype=torch.float16, device=DEV))


def test_refused_configurations():
    with pytest.raises(ValueError):
        tiny(0, 0)
    with pytest.raises(ValueError):
        tiny(None, 4)
    with pytest.raises(ValueError):
        attention.attention_for_request(
            torch.zeros(1, 4, 64, dtype=torch.float16, device=DEV), cache_with_a_row(), 0, "a", 5,
            torch.tensor([4], device=DEV), window=-1)


def cache_with_a_row():
    cache = PagedKVCache(CacheLayout(1, 4, 16, 2, 64), device=DEV)
    cache.reserve("a", 5)
    return cache
