"""CPU: a workspace on another device, or whose bytes are not side by side, is refused before the
library is called.  The tensors are stand-ins that say they are on a GPU; no call reaches one."""
from __future__ import annotations

import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flexengine_amd import _lib, ops

F16 = torch.float16


@pytest.fixture
def calls(monkeypatch):
    if not _lib.LIB_PATH.exists():
        from flexengine_amd import build
        build.build()
    seen = []
    monkeypatch.setattr(ops._lib, "call", lambda name, *args: seen.append(name))
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    with FakeTensorMode(), warnings.catch_warnings():
        warnings.simplefilter("ignore")   # addresses of stand-ins
        yield seen


def ints(*shape):
    return torch.empty(shape, dtype=torch.int32, device="cuda:0")


def call(op, kind, ws):
    q = torch.empty(2, 4, 64, dtype=F16, device="cuda:0")
    if kind == "kv4":
        pool = ops.Kv4Pool(torch.empty(4, 2, 16, 32, dtype=torch.uint8, device="cuda:0"),
                           torch.empty(4, 2, 16, 2, dtype=torch.uint8, device="cuda:0"), F16)
    else:
        pool = torch.empty(4, 16, 2, 64, dtype=F16, device="cuda:0")
    kw = dict(workspace=ws) | (dict(window=8, sinks=1) if kind == "window" else {})
    if op == "decode":
        return ops.paged_decode(q, pool, pool, ints(2, 3), ints(2), **kw)
    if op == "prefill":
        return ops.prefill_paged(q, pool, pool, ints(2, 3), ints(3), ints(2), 2, **kw)
    return ops.paged_decode_shared_prefix(q, pool, pool, ints(2, 3), ints(2), ints(2), ints(1), **kw)


OPS = [("decode", "plain"), ("decode", "window"), ("decode", "kv4"), ("prefill", "plain"),
       ("prefill", "window"), ("prefill", "kv4"), ("shared", "plain")]


@pytest.mark.parametrize("op,kind", OPS)
def test_workspaces_elsewhere_or_in_pieces_are_refused(calls, op, kind):
    size = 1 << 24
    for bad in (torch.empty(size, dtype=torch.uint8),
                torch.empty(size, dtype=torch.uint8, device="cuda:1"),
                torch.empty(size, 2, dtype=torch.uint8, device="cuda:0")[:, 0],
                torch.empty(1, dtype=torch.uint8, device="cuda:0").expand(size)):
        with pytest.raises(ValueError):
            call(op, kind, bad)
        assert not calls
    call(op, kind, torch.empty(size, dtype=torch.uint8, device="cuda:0"))
    assert len(calls) == 1
