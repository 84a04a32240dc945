"""GPU: 4-bit pools whose dims lie in another order or apart -- page writes, gather, decode and
prefill give what they give on dense pools, bit for bit, and write nothing between the rows."""
from __future__ import annotations

import pytest
import torch

from flexengine_amd import ops
from tests import span_ref as R
from tests.test_gpu_span import BF16, DEV, F16, Pools, gen, paged, packed, special_rows
from tests.test_gpu_span_prefill import Step

pytestmark = pytest.mark.gpu
FILL = 0x5A
# memory orders of blocks, heads, tokens: of the codes and of the scales; bytes between the rows
LAYOUTS = [("bth", "bth", 0), ("bth", "bht", 0), ("hbt", "tbh", 0), ("tbh", "hbt", 32), ("bht", "bht", 64)]


class Relaid:
    """A dense pool's bytes in another layout, FILL between the rows."""

    def __init__(self, pool, layout):
        self.memory, views = [], []
        for x, order, gap in ((pool.codes, layout[0], layout[2]), (pool.scales, layout[1], layout[2] // 16)):
            size = dict(zip("bht", x.shape))
            mem = torch.full([size[c] for c in order] + [x.shape[3] + gap], FILL, dtype=torch.uint8, device=DEV)
            view = mem.permute([order.index(c) for c in "bht"] + [3])[..., :x.shape[3]]
            view.copy_(x)
            self.memory.append((mem, x.shape[3]))
            views.append(view)
        self.pool = ops.Kv4Pool(*views, pool.dtype)

    def gaps_are_as_they_were(self):
        return all((mem[..., n:] == FILL).all() for mem, n in self.memory)


def same(pool, dense):
    return torch.equal(pool.codes, dense.codes) and torch.equal(pool.scales, dense.scales)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hkv,d,bs", [(2, 128, 16), (3, 96, 8), (1, 32, 4), (8, 64, 32), (2, 256, 16)])
def test_writes_and_gather(layout, dt, hkv, d, bs):
    lens, new = [1, 17, 0, 40, 33], [1, 5, 0, 40, 2]
    tables, nb = paged(lens, bs, 3, 5)
    tabs, ctx = tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    offs = torch.tensor([sum(new[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
    ends = torch.tensor([sum(lens[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
    k = special_rows(sum(new), hkv, d, dt, 6).to(DEV)
    v = torch.randn(k.shape, generator=gen(7)).to(dt).to(DEV)
    one = torch.randn(5, hkv, d, generator=gen(8)).to(dt).to(DEV)
    dense = [ops.Kv4Pool.empty((nb, bs, hkv, d), dt) for _ in range(2)]
    laid = [Relaid(p, layout) for p in dense]
    slot = torch.tensor([nb - 1, 0, -1], dtype=torch.int32, device=DEV)
    at = torch.tensor([bs - 1, 1, 0], dtype=torch.int32, device=DEV)
    got = []
    for pair in (dense, [x.pool for x in laid]):
        ops.write_kv_ragged(k, v, *pair, tabs, offs, ctx)
        ops.write_kv_decode(one, 2 * one, *pair, tabs, ctx)
        ops.write_kv(one[:3], one[2:], *pair, slot, at)
        got.append(ops.gather_kv(*pair, tabs, ctx, ends, sum(lens)))
    for x, p in zip(laid, dense):
        assert same(x.pool, p) and x.gaps_are_as_they_were()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(12, 2, 128, 16), (14, 2, 64, 32), (34, 2, 96, 16), (6, 2, 160, 16),
                                         (8, 1, 256, 16)])
def test_decode_with_and_without_new_rows(layout, dt, hq, hkv, d, bs):
    p = Pools([1, 70, 0, 500, 129, 16], bs, hkv, d, dt, 4, 0, 0, 22)
    laid = [Relaid(x, layout) for x in (p.kp, p.vp)]
    q = torch.randn(6, hq, d, generator=gen(1)).to(dt).to(DEV)
    new = torch.randn(6, hkv, d, generator=gen(2)).to(dt).to(DEV)
    for kw in (dict(), dict(window=90, sinks=5), dict(target_splits=1), dict(k_new=new, v_new=2 * new),
               dict(k_new=2 * new, v_new=new, window=90, sinks=5)):
        want = ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, **kw)
        got = ops.paged_decode(q, laid[0].pool, laid[1].pool, p.tabs, p.ctx, **kw)
        assert torch.isfinite(want).all() and torch.equal(got, want)
    for x, dense in zip(laid, (p.kp, p.vp)):
        assert same(x.pool, dense) and x.gaps_are_as_they_were()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(12, 2, 128, 16), (14, 2, 64, 32), (16, 4, 96, 64), (6, 2, 160, 16),
                                         (8, 1, 256, 16)])
def test_prefill(layout, dt, hq, hkv, d, bs):
    for window, sinks in ((0, 0), (90, 5)):
        s = Step([(90, 40), (0, 3), (700, 5), (300, 75)], bs, hq, hkv, d, dt, 4, window, sinks, 32)
        want = s.run()
        s.check(want, rows=6)
        s.kp, s.vp = Relaid(s.kp, layout).pool, Relaid(s.vp, layout).pool
        assert torch.equal(s.run(), want)


def test_rows_past_32_bit_offsets_by_token():
    """Pools by token whose codes pass 2^32 bytes: the last blocks written, read back, attended."""
    nb, bs, hkv, d, n = 300000, 32, 8, 128, 100
    assert nb * bs * hkv * d // 2 > 1 << 32
    pair = [ops.Kv4Pool(torch.empty(nb, bs, hkv, d // 2, dtype=torch.uint8, device=DEV).transpose(1, 2),
                        torch.empty(nb, bs, hkv, d // 32, dtype=torch.uint8, device=DEV).transpose(1, 2), F16)
            for _ in range(2)]
    tabs = torch.tensor([[nb - 1, nb - 5, nb // 2 + 7, nb - 2]], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    offs = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(n, hkv, d, generator=gen(70 + i)).half() for i in range(2))
    ops.write_kv_ragged(k.to(DEV), v.to(DEV), *pair, tabs, offs, ctx)
    kd, vd = R.round4(k), R.round4(v)
    ko, vo = ops.gather_kv(*pair, tabs, ctx, offs, n)
    assert torch.equal(ko.double().cpu(), kd) and torch.equal(vo.double().cpu(), vd)
    q = torch.randn(n, 16, d, generator=gen(72)).half()
    got = ops.prefill_paged(q.to(DEV), *pair, tabs, offs, ctx, n)
    R.assert_close(got, *R.attend(q, kd, vd, torch.arange(n), 0, 0))
    one = ops.paged_decode(q[-1:].to(DEV), *pair, tabs, ctx)
    R.assert_close(one, *R.attend(q[-1:], kd, vd, torch.tensor([n - 1]), 0, 0))


def test_captured_calls_over_pools_by_token():
    p = Pools([900, 20, 333], 16, 2, 128, F16, 4, 0, 0, 28)
    laid = [Relaid(x, LAYOUTS[0]).pool for x in (p.kp, p.vp)]
    q = torch.randn(3, 12, 128, generator=gen(3)).half().to(DEV)
    kn = torch.randn(3, 2, 128, generator=gen(4)).half().to(DEV)
    step = lambda pair: ops.paged_decode(q, *pair, p.tabs, p.ctx, k_new=kn, v_new=kn, window=256, sinks=4)  # noqa: E731
    with ops.hold_workspaces():
        step(laid)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(laid)
        for i in range(4):
            q.copy_(torch.randn(3, 12, 128, generator=gen(40 + i)).half())
            kn.copy_(torch.randn(3, 2, 128, generator=gen(50 + i)).half())
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, step((p.kp, p.vp))) and same(laid[0], p.kp) and same(laid[1], p.vp)


def test_packed_rows_are_what_the_pool_holds():
    x = special_rows(11, 2, 64, F16, 9)
    codes, scales = packed(x[:, None].transpose(1, 2))      # [11, 2, 1, *]
    dense = ops.Kv4Pool(codes.contiguous().to(DEV), scales.contiguous().to(DEV), F16)
    laid = Relaid(dense, LAYOUTS[1]).pool
    tabs = torch.arange(11, dtype=torch.int32, device=DEV)[:, None]
    ctx, ends = torch.ones(11, dtype=torch.int32, device=DEV), torch.arange(12, dtype=torch.int32, device=DEV)
    a, b = ops.gather_kv(dense, dense, tabs, ctx, ends, 11)[0], ops.gather_kv(laid, laid, tabs, ctx, ends, 11)[1]
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
