"""GPU: the forms that only large calls over 4-bit pools take -- 256 rows a workgroup in the
prefill, two tiles at a time in the decode -- and prefills whose lengths do not fit their tables
or rows.  Sizes that reach them: tests/test_span_forms.py."""
from __future__ import annotations

import pytest
import torch

from flexengine_amd import ops
from tests import span_ref as R
from tests.test_gpu_span import BF16, DEV, F16, JUNK, Pools, check_decode, gen
from tests.test_gpu_span_prefill import TYPES, Step

pytestmark = pytest.mark.gpu

# (cached, new) chunks, query and KV heads of 128, block size, window (0: none), sinks
LONG = [([(0, 2305)], 48, 1, 16, 0, 0),
        ([(3001, 2305)], 48, 1, 32, 4000, 70),
        ([(500, 2101), (0, 1999)], 48, 1, 16, 0, 0),
        ([(2600, 2101), (9, 2003)], 40, 2, 64, 4001, 3)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("chunks,hq,hkv,bs,window,sinks", LONG)
def test_long_prompts_over_4_bit_pools(dt, chunks, hq, hkv, bs, window, sinks):
    s = Step(chunks, bs, hq, hkv, 128, dt, 4, window, sinks, 60)
    got = s.run()
    s.check(got, rows=24)
    assert torch.isfinite(got).all() and torch.equal(s.run(), got)
    # the last rows of each chunk: waves whose rows are not all there
    for b, (c, n) in enumerate(chunks):
        idx = torch.tensor([0, 1, n - 2, n - 1])
        o = s.offs_list[b]
        out, bound = R.attend(s.q[o + idx], s.k[b], s.v[b], c + idx, window, sinks)
        R.assert_close(got[o + idx.to(DEV)], out, bound, f"ends of {c}+{n}")
    s.kp, s.vp = (ops.Kv4Pool(p.codes.transpose(1, 2).contiguous().transpose(1, 2),
                              p.scales.transpose(1, 2).contiguous().transpose(1, 2), dt) for p in (s.kp, s.vp))
    assert torch.equal(s.run(), got)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_long_prompts_are_the_same_captured(dt):
    chunks, hq, hkv, bs, window, sinks = LONG[0]
    s = Step(chunks, bs, hq, hkv, 128, dt, 4, window, sinks, 61)
    q = s.q.to(DEV)

    def call():
        return ops.prefill_paged(q, s.kp, s.vp, s.tabs, s.offs, s.ctx, s.max_new)

    with ops.hold_workspaces():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(3):
            q.copy_(torch.randn(q.shape, generator=gen(62 + i)).to(dt))
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, call())


# contexts of one row, with a window (0: none) and sinks, whose waves walk 16 tiles and more
WALKS = [(1024, 0, 0), (1025, 0, 0), (1100, 0, 0), (1184, 0, 0), (3999, 0, 0), (3000, 1501, 37), (2777, 1203, 16)]


def walked_tiles(n, window, sinks):
    """16-key tiles that a decode of n tokens walks."""
    head = -(-sinks // 16) if window else 0
    first = max(0, n - window) // 16 if window else 0
    return -(-n // 16) - max(0, first - head)


@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (6, 2, 96, 32), (12, 2, 128, 16), (6, 1, 160, 16),
                                         (8, 1, 256, 32), (1, 1, 32, 16)])
def test_two_tiles_at_a_time(dt, hq, hkv, d, bs, new):
    for i, (n, window, sinks) in enumerate(WALKS):
        p = Pools([n], bs, hkv, d, dt, 4, window, sinks, 80 + i)
        check_decode(p, hq, d, window or None, sinks, new=new, splits=1, seed=90 + i)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (14, 2, 64)])
def test_two_tiles_at_a_time_in_pieces_of_many_rows(dt, hq, hkv, d):
    """Long and short rows of one call in pieces of 16 quads and more, joined."""
    lengths = [6000, 3, 4100, 0, 2200, 1025]
    p = Pools(lengths, 16, hkv, d, dt, 4, 0, 0, 88)
    check_decode(p, hq, d, None, 0, new=True, splits=6)
    q = torch.randn(6, hq, d, generator=gen(5)).to(dt).to(DEV)
    outs = [ops.paged_decode(q, p.kp, p.vp, p.tabs, p.ctx, target_splits=6) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dt,bits", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (6, 2, 128)])
def test_contexts_past_the_table_and_shorter_than_their_rows(dt, bits, hq, hkv, d):
    """A context past its table ends with it, one shorter than its rows counts as those rows, and
    the other sequences' rows are as they were."""
    chunks = [(10, 20), (76, 20), (0, 12), (0, 4), (40, 8)]   # the second fills six pages
    s = Step(chunks, 16, hq, hkv, d, dt, bits, 64, 3, 48)
    s.tabs = s.tabs[:, :6].contiguous()
    want = s.run()
    s.check(want)
    for ctx in ([30, 1 << 30, 12, 4, 48], [30, 97, 5, 0, 48], [30, 96, 12, -3, 48], [30, 2 ** 31 - 1, 11, 1, 48]):
        s.ctx = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        assert torch.equal(s.run(), want), ctx


@pytest.mark.parametrize("dt,bits", TYPES)
def test_rows_past_the_table_leave_the_others_as_they_were(dt, bits):
    """More rows than the table has tokens: no entry past the table's last is read, and the other
    sequences' rows are as they were."""
    s = Step([(3, 9), (0, 40), (0, 16), (11, 5)], 16, 4, 2, 64, dt, bits, 7, 2, 49)
    full = s.run()
    s.tabs = s.tabs[:, :1].contiguous()
    got = s.run()
    for a, b in ((0, 9), (49, 65), (65, 70)):
        assert torch.equal(got[a:b], full[a:b])
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dt,bits", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
def test_decode_behind_the_widest_table(dt, bits, window, sinks):
    """Tables of 262144 tokens, as a captured step's may be, over contexts of at most 3000: the split
    and the workspace are the table's, the entries past the contexts name no block."""
    if bits != 4 and not window:
        pytest.skip("the plain decode")
    p = Pools([1, 3000, 0, 17, 64, 1500, 333], 16, 2, 128, dt, bits, window, sinks, 89)
    wide = torch.full((7, 262144 // 16), JUNK, dtype=torch.int32, device=DEV)
    wide[:, :p.tabs.shape[1]] = p.tabs
    p.tabs = wide
    check_decode(p, 12, 128, window or None, sinks, new=True)
