"""GPU: ragged prefill under a window with sinks over 16-bit, 32-bit and 4-bit pools, against the
definition in 64 bits (tests/span_ref.py)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from flexengine_amd import _lib, ops
from tests import span_ref as R
from tests.test_gpu_span import BF16, DEV, F16, F32, JUNK, gen, packed

pytestmark = pytest.mark.gpu
TYPES = [(F16, 4), (BF16, 4), (F16, 16), (BF16, 16), (F32, 32)]


class Step:
    """Chunks (cached, new) over pools that hold NaN except for what some row of the chunk sees
    (keys that only other sequences or no one sees are NaN, their pages no blocks)."""

    def __init__(self, chunks, bs, hq, hkv, d, dt, bits, window, sinks, seed):
        self.chunks, self.bits, self.dt = chunks, bits, dt
        self.window, self.sinks = window, sinks
        g = gen(seed)
        lens = [c + n for c, n in chunks]
        pages = [-(-n // bs) for n in lens]
        nb = sum(pages) + 3
        perm = list(range(nb))
        random.Random(seed).shuffle(perm)
        width = max(pages, default=1) + 2
        tables = torch.full((len(chunks), width), JUNK, dtype=torch.int32)
        kp = torch.full((nb, bs, hkv, d), math.nan, dtype=dt)
        vp = torch.full((nb, bs, hkv, d), math.nan, dtype=dt)
        self.k, self.v, at = [], [], 0
        for b, (c, n) in enumerate(chunks):
            first = max(0, c - window + 1) if window else 0
            k = torch.randn(c + n, hkv, d, generator=g).to(dt)
            v = torch.randn(c + n, hkv, d, generator=g).to(dt)
            seen = [j for j in range(c + n) if n and (j >= first or j < sinks)]
            for page in {j // bs for j in seen}:
                tables[b, page] = perm[at + page]
            if seen:
                idx = torch.tensor(seen)
                blk = tables[b, idx // bs].long()
                kp[blk, idx % bs], vp[blk, idx % bs] = k[idx], v[idx]
            at += pages[b]
            self.k.append(k), self.v.append(v)
        if bits == 4:
            def pool(x):
                c, s = packed(x.transpose(1, 2))
                return ops.Kv4Pool(c.contiguous().to(DEV), s.contiguous().to(DEV), dt)
            self.kp, self.vp = pool(kp), pool(vp)
            self.k, self.v = [R.round4(x) for x in self.k], [R.round4(x) for x in self.v]
        else:
            self.kp, self.vp = kp.to(DEV), vp.to(DEV)
        self.tabs = tables.to(DEV)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.offs_list = [sum(n for _, n in chunks[:i]) for i in range(len(chunks) + 1)]
        self.offs = torch.tensor(self.offs_list, dtype=torch.int32, device=DEV)
        self.q = torch.randn(self.offs_list[-1], hq, d, generator=g).to(dt)
        self.max_new = max((n for _, n in chunks), default=1)

    def run(self, **kw):
        span = dict(window=self.window, sinks=self.sinks) if self.window else {}
        return ops.prefill_paged(self.q.to(DEV), self.kp, self.vp, self.tabs, self.offs, self.ctx,
                                 self.max_new, **span, **kw)

    def check(self, got=None, rows=None, scale=None):
        got = self.run(scale=scale) if got is None else got
        for b, (c, n) in enumerate(self.chunks):
            pick = range(n) if rows is None or n <= rows else sorted(random.Random(b).sample(range(n), rows))
            idx = torch.tensor(list(pick), dtype=torch.long)
            if not len(idx):
                continue
            o = self.offs_list[b]
            out, bound = R.attend(self.q[o + idx], self.k[b], self.v[b], c + idx, self.window,
                                  self.sinks, scale)
            R.assert_close(got[o + idx.to(DEV)], out, bound, f"chunk {b} of {c}+{n}")


CHUNKS = [(0, 1), (0, 0), (5, 1), (0, 70), (200, 33), (63, 64), (640, 7), (0, 129)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 3), (16, 4), (64, 64), (63, 65), (65, 1),
                                          (100, 150), (5000, 7)])
@pytest.mark.parametrize("dt,bits", TYPES)
def test_prefill_windows_and_chunks(dt, bits, window, sinks):
    if bits != 4 and not window:
        pytest.skip("the plain prefill")
    Step(CHUNKS, 16, 12, 2, 128, dt, bits, window, sinks, 31).check()


@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (8, 8, 128, 32), (1, 1, 32, 16), (16, 1, 96, 64),
                                         (34, 2, 128, 16), (6, 2, 160, 16), (8, 1, 256, 16), (71, 1, 64, 128)])
@pytest.mark.parametrize("dt,bits", TYPES)
def test_prefill_heads_dims_blocks(dt, bits, hq, hkv, d, bs):
    if bits == 32 and d > 128:
        pytest.skip("float32 windows take head dims up to 128")
    Step([(90, 40), (0, 3), (300, 75)], bs, hq, hkv, d, dt, bits, 90, 5, 32).check(rows=24)


@pytest.mark.parametrize("d", [8, 40, 72, 104, 120])
@pytest.mark.parametrize("dt,bits", [(F16, 16), (BF16, 16), (F32, 32)])
def test_prefill_odd_head_dims(dt, bits, d):
    Step([(33, 50), (0, 90)], 16, 6, 2, d, dt, bits, 50, 3, 33).check(rows=30)


@pytest.mark.parametrize("dt,bits", TYPES)
def test_prefill_few_rows_over_a_long_context_join_their_splits(dt, bits):
    s = Step([(6000, 3), (2500, 1), (90, 2)], 16, 4, 1, 64, dt, bits, 5200, 70, 34)
    got = s.run()
    s.check(got)
    for _ in range(3):
        assert torch.equal(s.run(), got)


@pytest.mark.parametrize("dt,bits", TYPES)
def test_prefill_of_many_rows(dt, bits):
    s = Step([(0, 1300), (700, 600)], 16, 16, 4, 64 if bits == 32 else 128, dt, bits, 333, 4, 35)
    s.check(rows=40)


def test_prefill_long_prompt_without_a_window():
    s = Step([(0, 2111)], 32, 8, 2, 128, F16, 4, 0, 0, 36)
    s.check(rows=60)


@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 16), (F32, 32)])
def test_prefill_many_short_sequences(dt, bits):
    r = random.Random(6)
    chunks = [(r.choice((0, r.randrange(60))), r.randrange(0, 9)) for _ in range(150)]
    Step(chunks, 16, 4, 2, 64, dt, bits, 20, 2, 37).check()


def test_rows_behind_the_last_sequence_stay():
    s = Step([(10, 20)], 16, 4, 2, 64, F16, 4, 8, 1, 38)
    q = torch.cat((s.q, s.q[:5])).to(DEV)
    out = torch.full_like(q, 7.0)
    ops.prefill_paged(q, s.kp, s.vp, s.tabs, s.offs, s.ctx, 20, window=8, sinks=1, out=out)
    s.check(out)
    assert (out[20:] == 7.0).all()


def test_prefill_large_scores():
    s = Step([(100, 60)], 16, 8, 2, 128, F16, 16, 64, 4, 39)
    s.check(scale=1.7)


def test_decode_and_one_row_chunks_agree():
    s = Step([(700, 1), (64, 1), (0, 1)], 16, 12, 2, 128, BF16, 4, 200, 6, 40)
    a = s.run()
    b = ops.paged_decode(s.q.to(DEV), s.kp, s.vp, s.tabs, s.ctx, window=200, sinks=6)
    s.check(a), s.check(b)


@pytest.mark.parametrize("bits", [4, 16])
def test_prefill_captured_and_replayed_between_eager_calls(bits):
    s = Step([(900, 20), (0, 64), (333, 5)], 16, 12, 2, 128, F16, bits, 256, 4, 41)
    q = s.q.to(DEV)

    def step():
        return ops.prefill_paged(q, s.kp, s.vp, s.tabs, s.offs, s.ctx, 64, window=256, sinks=4)

    with ops.hold_workspaces() as held:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    assert held
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen(60 + i)).half())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_prefill_on_two_streams_with_their_own_workspaces():
    s = Step([(3000, 9), (2500, 40)], 16, 12, 2, 128, BF16, 4, 0, 0, 42)
    want, q = s.run(), s.q.to(DEV)
    need = _lib.load().fe_span_prefill_workspace_size(2, q.shape[0], 12, 2, 128)
    runs = [(torch.cuda.Stream(), torch.zeros(need, dtype=torch.uint8, device=DEV)) for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for st, ws in runs:
            with torch.cuda.stream(st):
                outs.append(ops.prefill_paged(q, s.kp, s.vp, s.tabs, s.offs, s.ctx, 40, workspace=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_prefill_refusals_on_the_gpu():
    s = Step([(10, 20)], 16, 4, 2, 64, F16, 4, 0, 0, 43)
    for kw in (dict(window=0), dict(window=8, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            s.run(**kw)
    plan = ops.prefill_paged_plan(s.offs, s.ctx, 20, 4, 2, s.tabs.shape[1], 16)
    with pytest.raises(ValueError):
        s.run(plan=plan)
    with pytest.raises(_lib.FlexEngineAMDError):
        s.run(scale=-1.0)
    with pytest.raises(_lib.FlexEngineAMDError):
        s.run(workspace=torch.zeros(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        ops.prefill_paged(s.q.bfloat16().to(DEV), s.kp, s.vp, s.tabs, s.offs, s.ctx, 20)


@pytest.mark.parametrize("dt,bits,d", [(F32, 32, 96), (F32, 32, 128), (F16, 16, 72), (BF16, 4, 160), (F16, 16, 256)])
def test_prefill_splits_at_other_head_dims(dt, bits, d):
    s = Step([(4000, 9), (0, 2), (2990, 30)], 16, 6, 2, d, dt, bits, 2600, 20, 44)
    got = s.run()
    s.check(got, rows=12)
    assert torch.equal(s.run(), got)


def test_prefill_splits_of_many_kv_heads_fit_the_workspace():
    s = Step([(1500, 1)], 16, 96, 96, 8, F32, 32, 1200, 0, 45)
    s.check()


@pytest.mark.parametrize("dt,bits", TYPES)
def test_prefill_non_finite_keys_reach_who_sees_them_alone(dt, bits):
    """A NaN key reaches the rows that see it (V of a row that some row of a unit sees has to be
    finite: K's is NaN here), in the same chunk and in no other sequence."""
    chunks, window, sinks = [(100, 60), (100, 60)], 24, 4
    a, b = (Step(chunks, 16, 4, 2, 64, dt, bits, window, sinks, 46) for _ in range(2))
    bad = torch.ones(1, 2, 64, dtype=dt, device=DEV)
    keep = torch.zeros_like(bad)
    bad[..., 7] = math.nan
    at = 120
    ops.write_kv(bad, keep, a.kp, a.vp, a.tabs[0, at // 16].reshape(1),
                 torch.tensor([at % 16], dtype=torch.int32, device=DEV))
    ops.write_kv(keep, keep, b.kp, b.vp, b.tabs[0, at // 16].reshape(1),
                 torch.tensor([at % 16], dtype=torch.int32, device=DEV))
    got, want = a.run(), b.run()
    sees = torch.tensor([100 + i >= at and 100 + i - at < window for i in range(60)])
    assert torch.isnan(got[:60].cpu()[sees]).all()
    idx = torch.nonzero(~sees)[:, 0]
    R.assert_close(got[idx.to(DEV)], *R.attend(a.q[idx], a.k[0], a.v[0], 100 + idx, window, sinks))
    assert torch.equal(got[60:], want[60:]) and torch.isfinite(want).all()


def test_prefill_workspaces_elsewhere_are_refused():
    s = Step([(10, 20)], 16, 4, 2, 64, F16, 4, 8, 1, 47)
    with pytest.raises(ValueError):
        s.run(workspace=torch.zeros(1 << 24, dtype=torch.uint8))
    with pytest.raises(ValueError):
        ops.paged_decode(s.q[:1].to(DEV), s.kp, s.vp, s.tabs, s.ctx, window=8,
                         workspace=torch.zeros(1 << 24, dtype=torch.uint8))


def test_prefill_sequences_longer_than_their_tables_or_contexts_stay_in_bounds():
    """Offsets past total_q, contexts past the table and shorter than the chunk: rows of other
    sequences are as they were."""
    s = Step([(10, 20), (40, 8)], 16, 4, 2, 64, F16, 16, 8, 1, 48)
    want = s.run()
    offs = torch.tensor([0, 20, 400], dtype=torch.int32, device=DEV)
    got = ops.prefill_paged(s.q.to(DEV), s.kp, s.vp, s.tabs, offs, s.ctx, 20, window=8, sinks=1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 16), (F32, 32)])
@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_captured_calls_follow_lengths_offsets_and_tables(kind, dt, bits):
    """Replays of one graph after its lengths, offsets and tables changed in place, between eager
    calls of the same."""
    steps = [Step(chunks, 16, 12, 2, 64, dt, bits, 300, 4, 50 + i) for i, chunks in enumerate(
        ([(900, 20), (0, 64), (333, 6)], [(0, 1), (1000, 49), (700, 40)], [(500, 88), (20, 1), (0, 1)]))]
    width = max(s.tabs.shape[1] for s in steps)
    blocks = max(s.kp.shape[0] for s in steps)
    wide = [torch.full((3, width), JUNK, dtype=torch.int32, device=DEV) for _ in steps]
    for t, s in zip(wide, steps):
        t[:, :s.tabs.shape[1]] = s.tabs

    def parts(pool):
        return (pool.codes, pool.scales) if bits == 4 else (pool,)

    def grown(pool):
        x = [torch.zeros((blocks,) + t.shape[1:], dtype=t.dtype, device=DEV) for t in parts(pool)]
        return ops.Kv4Pool(*x, dt) if bits == 4 else x[0]

    kp, vp, tabs, ctx = grown(steps[0].kp), grown(steps[0].vp), wide[0].clone(), steps[0].ctx.clone()
    offs, q = steps[0].offs.clone(), steps[0].q.to(DEV)
    rows = q if kind == "prefill" else q[:3].contiguous()

    def load(i):
        for mine, theirs in ((kp, steps[i].kp), (vp, steps[i].vp)):
            for a, b in zip(parts(mine), parts(theirs)):
                a[:b.shape[0]].copy_(b)
        tabs.copy_(wide[i]), ctx.copy_(steps[i].ctx), offs.copy_(steps[i].offs)
        rows.copy_(steps[i].q[:rows.shape[0]])

    def call():
        if kind == "decode":
            return ops.paged_decode(rows, kp, vp, tabs, ctx, window=300, sinks=4)
        return ops.prefill_paged(rows, kp, vp, tabs, offs, ctx, 88, window=300, sinks=4)

    with ops.hold_workspaces() as held:
        load(0)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
    assert held
    for i in (1, 2, 0, 1):
        load(i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call())
        if kind == "prefill":
            steps[i].check(got, rows=8)


@pytest.mark.parametrize("dt,bits,window,sinks", [(F16, 4, 0, 0), (BF16, 16, 300000, 70), (F32, 32, 100000, 33)])
def test_contexts_of_hundreds_of_thousands_of_tokens(dt, bits, window, sinks):
    """Long tables over a few pages in turn: a prefill of three rows and a decode at the longest
    table that it takes."""
    n, d, bs, nb = 400_003, 32, 16, 64
    k = torch.randn(nb * bs, 1, d, generator=gen(60)).to(dt)
    v = torch.randn(nb * bs, 1, d, generator=gen(61)).to(dt)
    pools = []
    for x in (k, v):
        pages = x.view(nb, bs, 1, d)
        if bits == 4:
            c, s = packed(pages.transpose(1, 2))
            pools.append(ops.Kv4Pool(c.contiguous().to(DEV), s.contiguous().to(DEV), dt))
        else:
            pools.append(pages.to(DEV))
    if bits == 4:
        k, v = R.round4(k), R.round4(v)
    q = torch.randn(3, 2, d, generator=gen(62)).to(dt)
    span = dict(window=window, sinks=sinks) if window else {}

    def rows(m):
        return (torch.arange(m) // bs % nb) * bs + torch.arange(m) % bs

    tabs = (torch.arange(-(-n // bs), dtype=torch.int32) % nb)[None].to(DEV)
    offs = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    got = ops.prefill_paged(q.to(DEV), *pools, tabs, offs, torch.tensor([n], dtype=torch.int32, device=DEV), 3, **span)
    at = rows(n)
    R.assert_close(got, *R.attend(q, k[at], v[at], torch.arange(n - 3, n), window, sinks))
    m = 262_144
    tabs = (torch.arange(m // bs, dtype=torch.int32) % nb)[None].to(DEV)
    got = ops.paged_decode(q[:1].to(DEV), *pools, tabs, torch.tensor([m], dtype=torch.int32, device=DEV), **span)
    at = rows(m)
    R.assert_close(got, *R.attend(q[:1], k[at], v[at], torch.tensor([m - 1]), window, sinks))
    with pytest.raises(_lib.FlexEngineAMDError):
        longer = torch.zeros(1, m // bs + 1, dtype=torch.int32, device=DEV)
        ops.paged_decode(q[:1].to(DEV), *pools, longer, torch.tensor([m], dtype=torch.int32, device=DEV), **span)


@pytest.mark.parametrize("dt,bits", [(F16, 4), (F32, 32)])
def test_one_row_chunks_of_many_sequences_over_long_contexts(dt, bits):
    r = random.Random(7)
    s = Step([(r.randrange(800, 1500), 1) for _ in range(150)], 16, 4, 1, 64, dt, bits, 1300, 20, 51)
    got = s.run()
    s.check(got)
    assert torch.equal(s.run(), got)


@pytest.mark.parametrize("dt,bits", TYPES)
def test_non_finite_keys_in_a_split(dt, bits):
    """A NaN in a split's keys makes NaN of the rows that see it once the splits are joined."""
    s = Step([(3000, 4), (2900, 2)], 16, 4, 1, 64, dt, bits, 2500, 8, 52)
    want = s.run()
    bad = torch.full((1, 1, 64), math.nan, dtype=dt, device=DEV)
    ops.write_kv(bad, bad, s.kp, s.vp, s.tabs[0, 1600 // 16].reshape(1),
                 torch.zeros(1, dtype=torch.int32, device=DEV))
    got = s.run()
    assert torch.isnan(got[:4]).all() and torch.equal(got[4:], want[4:]) and torch.isfinite(want).all()
