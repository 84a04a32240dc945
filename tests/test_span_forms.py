"""CPU: the sizes of tests/test_gpu_span_forms.py reach the kernels that they are for."""
from __future__ import annotations

import re

import pytest
import torch

from flexengine_amd import _lib, ops
from flexengine_amd import build as B
from tests import test_gpu_span_forms as G
from tests.test_span_host import lib  # noqa: F401

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("chunks,hq,hkv,bs,window,sinks", G.LONG)
def test_long_prompts_take_256_rows(lib, chunks, hq, hkv, bs, window, sinks):  # noqa: F811
    total = sum(n for _, n in chunks)
    span = dict(window=window, sinks=sinks) if window else {}
    assert ops.span_prefill_rows(len(chunks), total, hq, hkv, 128, F16, kv4=True, **span) == 256
    # the last unit of a sequence has waves without rows, and others have all
    assert any(n * (hq // hkv) % 256 for _, n in chunks)


def test_other_prefills_do_not(lib):  # noqa: F811
    assert ops.span_prefill_rows(1, 2305, 48, 1, 128, F16, kv4=True, window=3999) == 128
    assert ops.span_prefill_rows(1, 2305, 48, 1, 96, F16, kv4=True) == 128
    assert ops.span_prefill_rows(2, 2305, 48, 1, 128, F16, kv4=True) == 128
    assert ops.span_prefill_rows(1, 2305, 48, 1, 128, F16, window=5000) == 128
    assert ops.span_prefill_rows(1, 2305, 48, 1, 128, F32, window=5000) == 16
    for bad in (dict(num_seqs=0), dict(total_q=0), dict(kv_heads=5), dict(dtype=F32, kv4=True), dict()):
        kw = dict(num_seqs=1, total_q=9, num_q_heads=12, kv_heads=2, head_dim=128, dtype=F16) | bad
        with pytest.raises(_lib.FlexEngineAMDError):
            ops.span_prefill_rows(**kw, window=8 if bad and "kv4" not in bad else None)


def test_long_walks_take_two_tiles_at_once():
    text = (B.CSRC_DIR / "span_decode.hip").read_text()
    least = int(re.search(r"constexpr int kPairTiles = (\d+);", text).group(1))
    for n, window, sinks in G.WALKS:
        tiles = G.walked_tiles(n, window, sinks)
        waves = [len(range(w, tiles, 4)) for w in range(4)]
        assert min(waves) >= least and max(waves) <= 64, (n, window, waves)
    counts = {len(range(w, G.walked_tiles(*c), 4)) % 2 for c in G.WALKS for w in range(4)}
    assert counts == {0, 1}
    # the new token in the first and in the second tile of a pair
    last = {(G.walked_tiles(*c) - 1) // 4 % 2 for c in G.WALKS}
    assert last == {0, 1}
