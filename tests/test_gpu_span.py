"""GPU: 4-bit page writes and gathers, and decode under a window with sinks over 16-bit, 32-bit
and 4-bit pools, against the definitions in 64 bits (tests/span_ref.py)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from flexengine_amd import _lib, ops
from tests import span_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
JUNK = (1 << 30) + 12345   # a table entry that names no block


def gen(seed):
    return torch.Generator().manual_seed(seed)


def paged(lengths, bs, spare, seed, hole=None):
    """(tables int32 [B, W], num_blocks): shuffled pages; entries past a length, and those that
    hole(b, page) says, name no block."""
    pages = [-(-n // bs) for n in lengths]
    nb = sum(pages) + spare
    perm = list(range(nb))
    random.Random(seed).shuffle(perm)
    width = max(max(pages, default=1), 1) + 1
    tables = torch.full((len(lengths), width), JUNK, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        for j in range(p):
            tables[b, j] = -7 if hole and hole(b, j) else perm[at + j]
        at += p
    return tables, nb


def special_rows(t, hkv, d, dt, seed):
    """Rows with the blocks where packing can go wrong."""
    x = torch.randn(t, hkv, d, generator=gen(seed)).to(dt)
    x[0] = 0
    if t > 1:
        x[1, :, ::2] = -0.0
    if t > 2:  # ties of every pair of neighbouring codes, at a scale of 2^-3
        ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5]) / 8
        x[2] = torch.cat((ties, -ties)).repeat(d // 16).to(dt)
        x[2, :, ::32] = 7.0 / 8
    if t > 3:
        x[3] = (torch.rand(hkv, d, generator=gen(seed + 1)) * 2.0 ** -22).to(dt)
    if t > 4:
        x[4, :, 3] = 65504.0 if dt == F16 else 3.0e38
    if t > 5:
        x[5, 0, 5] = math.inf
        x[5, -1, d - 1] = math.nan
    if t > 6:  # the borders between two scales
        x[6, :, 0] = 1.75
        x[6, :, 1:32] = x[6, :, 1:32].clamp(-1, 1)
    if t > 7:
        x[7, :, 0] = 1.7509765625 if dt == F16 else 1.7578125
        x[7, :, 1:32] = x[7, :, 1:32].clamp(-1, 1)
    return x


def packed(x):
    """The bytes of rows, [..., D/2] and [..., D/32]; a NaN block's codes are not compared."""
    code, scale = R.pack_rows(x)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale


def assert_row(codes, scales, want_codes, want_scales):
    assert torch.equal(scales, want_scales)
    keep = (want_scales != 255).repeat_interleave(16, -1)
    assert torch.equal(codes[keep], want_codes[keep])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hkv,d,bs", [(1, 32, 1), (2, 64, 16), (8, 128, 16), (3, 96, 8), (2, 256, 32)])
def test_slot_write_packs_rows_and_touches_nothing_else(dt, hkv, d, bs):
    t, nb = 11, 29
    k, v = special_rows(t, hkv, d, dt, 1), special_rows(t, hkv, d, dt, 2)
    # rows of a fused projection: heads contiguous, rows apart
    wide = torch.empty(t, 2 * hkv * d + 16, dtype=dt, device=DEV)
    kd = wide[:, :hkv * d].view(t, hkv, d)
    vd = wide[:, hkv * d + 8:2 * hkv * d + 8].view(t, hkv, d)
    kd.copy_(k), vd.copy_(v)
    kp, vp = (ops.Kv4Pool.empty((nb, bs, hkv, d), dt) for _ in range(2))
    for p in (kp, vp):
        p.codes.fill_(0xA5), p.scales.fill_(77)
    slots = random.Random(3).sample(range(nb * bs), t)
    block = torch.tensor([s // bs for s in slots], dtype=torch.int32)
    off = torch.tensor([s % bs for s in slots], dtype=torch.int32)
    block[8], block[9], off[10] = -1, nb, bs   # nowhere
    ops.write_kv(kd, vd, kp, vp, block.to(DEV), off.to(DEV))
    for pool, x in ((kp, k), (vp, v)):
        codes, scales = pool.codes.cpu(), pool.scales.cpu()
        wc, ws = packed(x)
        for i in range(8):
            b, o = int(block[i]), int(off[i])
            assert_row(codes[b, :, o], scales[b, :, o], wc[i], ws[i])
            codes[b, :, o], scales[b, :, o] = 0xA5, 77
        assert (codes == 0xA5).all() and (scales == 77).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hkv,d,bs", [(2, 64, 16), (8, 128, 32), (1, 160, 4)])
def test_decode_and_ragged_writes_then_gather(dt, hkv, d, bs):
    lens = [1, 17, 0, 40, 33]
    new = [1, 5, 0, 40, 2]
    tables, nb = paged(lens, bs, 3, 5)
    tabs, ctx = tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    offs = torch.tensor([sum(new[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
    kp, vp = (ops.Kv4Pool.empty((nb, bs, hkv, d), dt) for _ in range(2))
    k = special_rows(sum(new) + 2, hkv, d, dt, 6).to(DEV)   # two rows behind the last sequence
    v = torch.randn(k.shape, generator=gen(7)).to(dt).to(DEV)
    ops.write_kv_ragged(k, v, kp, vp, tabs, offs, ctx)
    want = {b: (torch.zeros(n, hkv, d, dtype=torch.float64), torch.zeros(n, hkv, d, dtype=torch.float64))
            for b, n in enumerate(lens)}
    for b, (n, m) in enumerate(zip(lens, new)):
        at = int(offs[b])
        want[b][0][n - m:] = R.round4(k[at:at + m].cpu())
        want[b][1][n - m:] = R.round4(v[at:at + m].cpu())
    # then one more token each by the decode form, at the last position
    k1 = torch.randn(5, hkv, d, generator=gen(8)).to(dt)
    ops.write_kv_decode(k1.to(DEV), (2 * k1).to(DEV), kp, vp, tabs, ctx)
    for b, n in enumerate(lens):
        if n:
            want[b][0][n - 1], want[b][1][n - 1] = R.round4(k1)[b], R.round4(2 * k1)[b]
    ends = torch.tensor([sum(lens[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
    ko, vo = ops.gather_kv(kp, vp, tabs, ctx, ends, sum(lens))
    assert ko.dtype == dt
    for got, j in ((ko, 0), (vo, 1)):
        exp = torch.cat([want[b][j] for b in range(5)])
        assert torch.equal(torch.nan_to_num(got.double().cpu(), nan=-9e9), torch.nan_to_num(exp, nan=-9e9))


class Pools:
    """Pools that hold NaN except for the rows that a decode of these lengths sees."""

    def __init__(self, lengths, bs, hkv, d, dt, bits, window, sinks, seed, cover=1):
        self.lengths, self.bits, self.dt = lengths, bits, dt
        first = lambda n: max(0, n - cover - window + 1) if window else 0  # noqa: E731
        seen = lambda n, j: j >= first(n) or j < min(sinks, n)  # noqa: E731
        self.tables, nb = paged(lengths, bs, 2, seed, hole=lambda b, page: not any(
            seen(lengths[b], j) for j in range(page * bs, min((page + 1) * bs, lengths[b]))))
        g = gen(seed)
        self.k = [torch.randn(n, hkv, d, generator=g).to(dt) for n in lengths]
        self.v = [torch.randn(n, hkv, d, generator=g).to(dt) for n in lengths]
        kp = torch.full((nb, bs, hkv, d), math.nan, dtype=dt)
        vp = torch.full((nb, bs, hkv, d), math.nan, dtype=dt)
        for b, n in enumerate(lengths):
            for j in range(n):
                if seen(n, j):
                    kp[self.tables[b, j // bs], j % bs] = self.k[b][j]
                    vp[self.tables[b, j // bs], j % bs] = self.v[b][j]
        if bits == 4:
            def pool(x):
                c, s = packed(x.transpose(1, 2))
                c = torch.where((s == 255).repeat_interleave(16, -1), torch.tensor(0x77, dtype=torch.uint8), c)
                return ops.Kv4Pool(c.contiguous().to(DEV), s.contiguous().to(DEV), dt)
            self.kp, self.vp = pool(kp), pool(vp)
            self.k, self.v = [R.round4(x) for x in self.k], [R.round4(x) for x in self.v]
        else:
            self.kp, self.vp = kp.to(DEV), vp.to(DEV)
        self.tabs = self.tables.to(DEV)
        self.ctx = torch.tensor(lengths, dtype=torch.int32, device=DEV)


LENGTHS = [1, 0, 15, 16, 17, 64, 100, 333, 1000]
SPANS = [(None, 0), (1, 0), (1, 1), (16, 4), (17, 0), (64, 16), (63, 17), (100, 33), (300, 200),
         (4096, 4), (1 << 31, 1 << 31)]


def check_decode(p, hq, d, window, sinks, new=False, strided=False, splits=0, seed=11, scale=None):
    b = len(p.lengths)
    q = torch.randn(b, hq, d, generator=gen(seed)).to(p.dt)
    qd = q.to(DEV)
    if strided:
        qd = torch.cat((qd.flatten(1), torch.zeros(b, 8, dtype=p.dt, device=DEV)), 1)[:, :hq * d].view(b, hq, d)
    hkv = p.k[0].shape[1]
    kn = vn = None
    if new:
        kn = torch.randn(b, hkv, d, generator=gen(seed + 1)).to(p.dt)
        vn = torch.randn(b, hkv, d, generator=gen(seed + 2)).to(p.dt)
    span = {} if window is None else dict(window=window, sinks=sinks)
    got = ops.paged_decode(qd, p.kp, p.vp, p.tabs, p.ctx, target_splits=splits, scale=scale,
                           k_new=None if kn is None else kn.to(DEV),
                           v_new=None if vn is None else vn.to(DEV), **span).cpu()
    for i, n in enumerate(p.lengths):
        if n == 0:
            assert (got[i] == 0).all()
            continue
        k, v = p.k[i], p.v[i]
        if new:
            k, v = k.clone(), v.clone()
            k[n - 1] = R.round4(kn[i]) if p.bits == 4 else kn[i]
            v[n - 1] = R.round4(vn[i]) if p.bits == 4 else vn[i]
        out, bound = R.attend(q[i:i + 1], k, v, torch.tensor([n - 1]), window or 0, sinks, scale)
        R.assert_close(got[i:i + 1], out, bound, f"length {n}")
    if new:  # the rows are in the pools, in the rows' places
        tail = torch.tensor([[p.tables[i, max(n - 1, 0) // p.kp.shape[1]]] for i, n in enumerate(p.lengths)],
                            dtype=torch.int32)
        held = [(n - 1) % p.kp.shape[1] + 1 if n else 0 for n in p.lengths]
        ends = [sum(held[:i]) for i in range(b + 1)]
        ko, vo = ops.gather_kv(p.kp, p.vp, tail.clamp(0, p.kp.shape[0] - 1).to(DEV),
                               torch.tensor(held, dtype=torch.int32, device=DEV),
                               torch.tensor(ends, dtype=torch.int32, device=DEV), ends[-1])
        for i, n in enumerate(p.lengths):
            if n:
                for o, x in ((ko, kn), (vo, vn)):
                    exp = R.round4(x[i]) if p.bits == 4 else x[i].double()
                    assert torch.equal(o[ends[i + 1] - 1].double().cpu(), exp)


@pytest.mark.parametrize("window,sinks", SPANS)
@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 4), (F16, 16), (BF16, 16), (F32, 32)])
def test_decode_windows_and_lengths(dt, bits, window, sinks):
    if bits != 4 and window is None:
        pytest.skip("the plain decode")
    p = Pools(LENGTHS, 16, 2, 128, dt, bits, window or 0, sinks, 21)
    check_decode(p, 12, 128, window, sinks)


@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (8, 8, 128, 32), (1, 1, 32, 16), (16, 1, 96, 64),
                                         (34, 2, 128, 16), (6, 2, 160, 16), (8, 1, 256, 16), (71, 1, 64, 128)])
@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 4), (F16, 16), (BF16, 16), (F32, 32)])
def test_decode_heads_dims_blocks_with_new_rows(dt, bits, hq, hkv, d, bs):
    if bits == 32 and d > 128:
        pytest.skip("float32 windows take head dims up to 128")
    p = Pools([1, 70, 0, 500, 129, 16], bs, hkv, d, dt, bits, 90, 5, 22)
    check_decode(p, hq, d, 90, 5, new=True, strided=True)


@pytest.mark.parametrize("d", [8, 40, 72, 104, 120])
@pytest.mark.parametrize("dt,bits", [(F16, 16), (BF16, 16), (F32, 32)])
def test_decode_odd_head_dims(dt, bits, d):
    p = Pools([33, 200], 16, 2, d, dt, bits, 50, 3, 23)
    check_decode(p, 6, d, 50, 3, new=True)


@pytest.mark.parametrize("splits", [1, 7, 64])
@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 16), (F32, 32)])
def test_decode_splits_agree_and_repeat(dt, bits, splits):
    p = Pools([5000, 3, 2500], 16, 1, 64, dt, bits, 4000, 40, 24)
    check_decode(p, 4, 64, 4000, 40, splits=splits)
    q = torch.randn(3, 4, 64, generator=gen(1)).to(dt).to(DEV)
    outs = [ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, window=4000, sinks=40, target_splits=splits)
            for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_window_past_every_context_is_the_plain_decode_to_rounding():
    p = Pools([700, 31, 64], 16, 2, 128, F16, 16, 0, 0, 25)
    q = torch.randn(3, 12, 128, generator=gen(2)).half().to(DEV)
    a = ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx)
    b = ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, window=701)
    # each is within 2^-11 of its values of the same number, twice (output, probabilities)
    assert (a.double() - b.double()).abs().max() <= 4 * 2.0 ** -11 * 4.5


def test_decode_many_short_rows_and_more_rows_than_a_wave():
    lens = [random.Random(4).randrange(0, 90) for _ in range(150)]
    p = Pools(lens, 16, 2, 64, BF16, 4, 20, 2, 26)
    check_decode(p, 4, 64, 20, 2, new=True)


def test_large_scores_and_scale():
    p = Pools([300], 16, 1, 128, F16, 4, 128, 4, 27)
    check_decode(p, 8, 128, 128, 4, scale=1.7)


@pytest.mark.parametrize("bits", [4, 16])
def test_decode_captured_and_replayed_between_eager_calls(bits):
    p = Pools([900, 20, 333], 16, 2, 128, F16, bits, 256, 4, 28)
    q = torch.randn(3, 12, 128, generator=gen(3)).half().to(DEV)
    kn = torch.randn(3, 2, 128, generator=gen(4)).half().to(DEV)

    def step():
        return ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, k_new=kn, v_new=kn, window=256, sinks=4)

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
        q.copy_(torch.randn(3, 12, 128, generator=gen(40 + i)).half())
        kn.copy_(torch.randn(3, 2, 128, generator=gen(50 + i)).half())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_decode_on_two_streams_with_their_own_workspaces():
    p = Pools([4000, 3500, 77], 16, 2, 128, BF16, 4, 0, 0, 29)
    q = torch.randn(3, 12, 128, generator=gen(5)).to(BF16).to(DEV)
    want = ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx)
    need = _lib.load().fe_span_decode_workspace_size(3, 12, 2, 128, p.tabs.shape[1] * 16, 0)
    runs = [(torch.cuda.Stream(), torch.zeros(need, dtype=torch.uint8, device=DEV)) for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, ws in runs:
            with torch.cuda.stream(s):
                outs.append(ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, workspace=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def high_rows(nb, bs, hkv, d, dt, bits, blocks, k, v):
    """Pools of nb blocks, nothing but `blocks` filled: with the rows k, v [len(blocks) * bs, hkv, d]."""
    slots = [t.repeat_interleave(bs) if i == 0 else t.repeat(len(blocks)) for i, t in enumerate(
        (torch.tensor(blocks, dtype=torch.int32, device=DEV), torch.arange(bs, dtype=torch.int32, device=DEV)))]
    if bits == 4:
        make = lambda: ops.Kv4Pool(torch.empty(nb, hkv, bs, d // 2, dtype=torch.uint8, device=DEV),  # noqa: E731
                                   torch.empty(nb, hkv, bs, d // 32, dtype=torch.uint8, device=DEV), dt)
    else:
        make = lambda: torch.empty(nb, bs, hkv, d, dtype=dt, device=DEV)  # noqa: E731
    kp, vp = make(), make()
    ops.write_kv(k.to(DEV), v.to(DEV), kp, vp, *slots)
    return kp, vp


@pytest.mark.parametrize("dt,bits,nb", [(F16, 16, 140000), (F32, 32, 70000), (BF16, 4, 300000)])
def test_pools_past_32_bit_offsets(dt, bits, nb):
    """The last blocks of pools whose elements (4-bit: bytes) pass 2^32 (fp32: 2^31): written in
    every way, gathered, attended by a decode with a new row and by a prefill."""
    bs, hkv, d, hq, n = 32, 8, 128, 16, 100
    assert nb * bs * hkv * d >> (1 if bits == 4 else 0) >= 1 << (31 if bits == 32 else 32)
    blocks = [nb - 1, nb - 5, nb // 2 + 7, nb - 2]
    k = torch.randn(4 * bs, hkv, d, generator=gen(70)).to(dt)
    v = torch.randn(4 * bs, hkv, d, generator=gen(71)).to(dt)
    kp, vp = high_rows(nb, bs, hkv, d, dt, bits, blocks, k, v)
    tabs = torch.tensor([blocks], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    offs = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    ops.write_kv_ragged(k[60:n].to(DEV), v[60:n].to(DEV), kp, vp, tabs, offs, ctx)
    ops.write_kv_decode(k[n - 1:n].to(DEV), v[n - 1:n].to(DEV), kp, vp, tabs, ctx)
    hold = R.round4 if bits == 4 else (lambda x: x.double())
    ko, vo = ops.gather_kv(kp, vp, tabs, ctx, torch.tensor([0, n], dtype=torch.int32, device=DEV), n)
    assert torch.equal(ko.double().cpu(), hold(k[:n])) and torch.equal(vo.double().cpu(), hold(v[:n]))
    q = torch.randn(40, hq, d, generator=gen(72)).to(dt)
    got = ops.prefill_paged(q.to(DEV), kp, vp, tabs, offs, ctx, 40, window=50, sinks=3)
    R.assert_close(got, *R.attend(q, hold(k[:n]), hold(v[:n]), torch.arange(60, n), 50, 3))
    k[n], v[n] = k[0].clone(), v[3].clone()
    got = ops.paged_decode(q[:1].to(DEV), kp, vp, tabs, ctx + 1, k_new=k[n:n + 1].to(DEV),
                           v_new=v[n:n + 1].to(DEV), window=70, sinks=5)
    R.assert_close(got, *R.attend(q[:1], hold(k[:n + 1]), hold(v[:n + 1]), torch.tensor([n]), 70, 5))
    ko, vo = ops.gather_kv(kp, vp, tabs, ctx + 1, torch.tensor([0, n + 1], dtype=torch.int32, device=DEV), n + 1)
    assert torch.equal(ko.double().cpu(), hold(k[:n + 1])) and torch.equal(vo.double().cpu(), hold(v[:n + 1]))


@pytest.mark.parametrize("s", [512, 513, 700])
def test_ragged_writes_and_gathers_of_many_sequences(s):
    r = random.Random(s)
    lens = [r.randrange(0, 6) for _ in range(s)]
    new = [r.randrange(0, n + 1) for n in lens]
    tables, nb = paged(lens, 4, 1, s)
    tabs, ctx = tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    offs = torch.tensor([sum(new[:i]) for i in range(s + 1)], dtype=torch.int32, device=DEV)
    kp, vp = (ops.Kv4Pool.empty((nb, 4, 1, 32), F16) for _ in range(2))
    k = torch.randn(sum(new), 1, 32, generator=gen(73)).half()
    ops.write_kv_ragged(k.to(DEV), (-k).to(DEV), kp, vp, tabs, offs, ctx)
    ends = torch.tensor([sum(lens[:i]) for i in range(s + 1)], dtype=torch.int32, device=DEV)
    ko, vo = ops.gather_kv(kp, vp, tabs, ctx, ends, sum(lens))
    want, at = [], 0
    for n, m in zip(lens, new):
        want += [torch.zeros(n - m, 1, 32, dtype=torch.float64), R.round4(k[at:at + m])]
        at += m
    want = torch.cat(want)
    assert torch.equal(ko.double().cpu(), want) and torch.equal(vo.double().cpu(), -want)


@pytest.mark.parametrize("dt,bits", [(F16, 4), (BF16, 16), (F32, 32)])
@pytest.mark.parametrize("splits", [1, 16])
def test_decode_non_finite_rows_are_nan_for_who_sees_them_alone(dt, bits, splits):
    """A row's NaN or infinity reaches the queries of its sequence that see it, no others."""
    n, window, sinks = 405, 64, 4
    p = Pools([n, n, n, n], 16, 1, 64, dt, bits, 0, 0, 74)
    want = Pools([n, n, n, n], 16, 1, 64, dt, bits, 0, 0, 74)
    bad = torch.ones(1, 1, 64, dtype=dt, device=DEV)
    bad[0, 0, 7] = math.nan

    def put(b, j, pool_k):
        rows = [torch.ones_like(bad), torch.ones_like(bad)]
        rows[0 if pool_k else 1] = bad
        blk = p.tabs[b, j // 16].reshape(1)
        ops.write_kv(*rows, p.kp, p.vp, blk, torch.tensor([j % 16], dtype=torch.int32, device=DEV))

    put(0, 350, True)        # seen: its K
    put(1, 2, False)         # seen: a sink's V
    put(2, 340, True)        # just before the window (341 on), in its first tile
    put(2, 336, False)
    put(3, 4, False)         # behind the sinks, in their tile
    q = torch.randn(4, 8, 64, generator=gen(75)).to(dt).to(DEV)
    run = lambda s: ops.paged_decode(q, s.kp, s.vp, s.tabs, s.ctx, window=window,  # noqa: E731
                                     sinks=sinks, target_splits=splits)
    got, ref = run(p), run(want)
    assert torch.equal(got[2:], ref[2:]) and torch.isfinite(ref).all()
    assert torch.isnan(got[0]).all()
    seen = torch.isnan(got[1])   # of the row, or the 4-bit row's block
    assert seen[:, 7].all() and seen[:, :32].all() == (bits == 4) and not seen[:, 32:].any()


@pytest.mark.parametrize("dt,bits", [(F16, 4), (F16, 16), (F32, 32)])
def test_decode_lengths_past_the_table_end_at_it(dt, bits):
    p = Pools([64, 40], 16, 2, 64, dt, bits, 0, 0, 76)
    width = 3                         # tables of 48 tokens
    tabs = p.tabs[:, :width].contiguous()
    q = torch.randn(2, 4, 64, generator=gen(77)).to(dt).to(DEV)
    long = torch.tensor([1 << 30, 40], dtype=torch.int32, device=DEV)
    cut = torch.tensor([48, 40], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.paged_decode(q, p.kp, p.vp, tabs, long, window=20, sinks=2),
                       ops.paged_decode(q, p.kp, p.vp, tabs, cut, window=20, sinks=2))
    neg = torch.tensor([-5, 40], dtype=torch.int32, device=DEV)
    got = ops.paged_decode(q, p.kp, p.vp, tabs, neg, window=20, sinks=2)
    assert (got[0] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("dt,bits", [(F16, 4), (F16, 16), (F32, 32)])
def test_decode_new_rows_without_a_page_are_not_written(dt, bits):
    p = Pools([33, 33], 16, 2, 64, dt, bits, 0, 0, 78)
    tabs = p.tabs.clone()
    tabs[0, 2] = JUNK                 # the new token's page
    q = torch.randn(2, 4, 64, generator=gen(79)).to(dt).to(DEV)
    kn = torch.randn(2, 2, 64, generator=gen(80)).to(dt).to(DEV)
    raw = lambda: [t.clone() for x in (p.kp, p.vp) for t in ((x.codes, x.scales) if bits == 4 else (x,))]  # noqa: E731
    before = raw()
    blk = int(p.tabs[1, 2])
    a = ops.paged_decode(q, p.kp, p.vp, tabs, p.ctx, k_new=kn, v_new=kn, window=30, sinks=2)
    for x, y in zip(before, raw()):
        same = (x.view(torch.uint8) == y.view(torch.uint8)).flatten(1).all(1)
        same[blk] = True
        assert same.all()
    assert torch.isfinite(a[1]).all()


@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_a_workspace_made_in_a_capture_is_the_graphs_alone(kind):
    p = Pools([3000], 16, 2, 128, F16, 4, 0, 0, 81)
    q = torch.randn(1, 12, 128, generator=gen(82)).half().to(DEV)
    offs = torch.tensor([0, 1], dtype=torch.int32, device=DEV)

    def step():
        if kind == "decode":
            return ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, window=2500, sinks=4)
        return ops.prefill_paged(q, p.kp, p.vp, p.tabs, offs, p.ctx, 1, window=2500, sinks=4)

    key = ("cuda", 0, "span_" + kind)
    step()
    kept = ops._WORKSPACES.pop(key)
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with ops.hold_workspaces() as held, torch.cuda.graph(graph):
            a, b = step(), step()
        assert len(held) == 2 and key not in ops._WORKSPACES
        for i in range(4):
            q.copy_(torch.randn(1, 12, 128, generator=gen(90 + i)).half())
            want = step()             # before the first replay too
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(step(), want)
    finally:
        ops._WORKSPACES[key] = kept


def test_refusals_on_the_gpu():
    p = Pools([40], 16, 2, 64, F16, 4, 0, 0, 30)
    q = torch.zeros(1, 4, 64, dtype=F16, device=DEV)
    call = lambda **kw: ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, **kw)  # noqa: E731
    for kw in (dict(window=0), dict(window=-3), dict(window=8, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(window=1.5)
    with pytest.raises(ValueError):   # a 4-bit pool beside a 16-bit one
        ops.paged_decode(q, p.kp, torch.zeros(1, 16, 2, 64, dtype=F16, device=DEV), p.tabs, p.ctx)
    with pytest.raises(ValueError):   # another type than the rows'
        ops.paged_decode(q.bfloat16(), p.kp, p.vp, p.tabs, p.ctx)
    with pytest.raises(ValueError):
        ops.paged_decode_shared_prefix(q, p.kp, p.vp, p.tabs, p.ctx, p.ctx, p.ctx)
    plan = ops.paged_decode_plan(p.tabs, p.ctx, 4, 2, 16)
    with pytest.raises(ValueError):
        call(plan=plan)
    with pytest.raises(_lib.FlexEngineAMDError):
        call(workspace=torch.zeros(1 << 10, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        ops.Kv4Pool.empty((4, 16, 2, 48), F16)
    with pytest.raises(ValueError):
        ops.Kv4Pool.empty((4, 16, 2, 64), F32)
    small = ops.Kv4Pool.empty((4, 8, 2, 64), F16)   # pages of 8 tokens
    with pytest.raises(_lib.FlexEngineAMDError):
        ops.paged_decode(q, small, small, p.tabs, p.ctx)
