"""Attention over long contexts: a KV cache held in 4 bits, and a sliding window with sinks.

The operators, as timed cases over the package's public entry points:

* 4-bit cache: rows are stored as blocks of 32 values with one power-of-two scale (e2m1 codes,
  e8m0 scales); ragged and single-token page writes, the gather back to 16 bits, the
  single-token decode (with the new token's write in the same call) and the ragged prefill.
* window: a query at position p sees the keys j <= p with p - j < window, and the first `sinks`
  keys of its sequence whatever the distance; decode and prefill over 16-bit, 32-bit and
  4-bit pools.

Kinds of case (`case["kind"]`):

* store:   page write of the chunks of a ragged step, and the gather of the whole contexts.
* append:  page write of one token per row, and the gather of the pages written to.
* decode:  the attention of one decode step over several layers.
* step:    the same with each layer's page write in the attention call, and the last pages.
* prefill: the attention of a ragged prefill step.

`bits` is what a cached value takes: 4, 16 (of `dtype`) or 32.  Where `own` is false, run()
computes the definition with elementary operations in 32 bits; where it is true it makes the
package's calls.  Head shapes, block sizes and lengths are those of the repository's workloads
and tests (12/2/128, 14/2/64) and a generic 32/8/128 and 16/4/96.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
HEADS = ((12, 2, 128), (14, 2, 64), (32, 8, 128), (16, 4, 96))
# the scale exponents of a 4-bit block: values are multiples of 2^-24 and, in float16, finite
E_LOW, E_HIGH = -23, {"float16": 13, "bfloat16": 125}


def listed():
    return [
        # the new tokens of a small server's step put into a 4-bit cache: the smallest call
        dict(name="append_small", kind="append", rows=8, lo=16, hi=512, hq=14, hkv=2, d=64,
             dtype="float16", bits=4, block=16, window=0, sinks=0, layers=1, sizes=1),
        # the prompts of a prefill step stored in 4 bits and read back: the write's throughput
        dict(name="store_prompts", kind="store", chunks=4, new_lo=800, new_hi=2500, cached_hi=0,
             hq=32, hkv=8, d=128, dtype="bfloat16", bits=4, block=16, window=0, sinks=0,
             layers=1, sizes=2),
        # one chat request's next token over a 4-bit cache: latency
        dict(name="token4", kind="decode", rows=1, lo=512, hi=512, hq=12, hkv=2, d=128,
             dtype="float16", bits=4, block=16, window=0, sinks=0, layers=1, sizes=3),
        # a busy server's decode step over a 4-bit cache: 64 rows, mixed contexts, with the
        # page write of the new tokens
        dict(name="step4_mixed", kind="step", rows=64, lo=128, hi=4096, hq=12, hkv=2, d=128,
             dtype="float16", bits=4, block=16, window=0, sinks=0, layers=2, sizes=4),
        # long-context decode, larger pages: the most K/V that one step reads here
        dict(name="decode4_long", kind="decode", rows=37, lo=2048, hi=16384, hq=32, hkv=8, d=128,
             dtype="bfloat16", bits=4, block=32, window=0, sinks=0, layers=2, sizes=5),
        # continuous batching: four prompt chunks over contexts cached in 4 bits
        dict(name="chunks4", kind="prefill", chunks=4, new_lo=256, new_hi=500, cached_hi=3000,
             hq=12, hkv=2, d=128, dtype="float16", bits=4, block=16, window=0, sinks=0, layers=1,
             sizes=6),
        # one long prompt at once over a 4-bit cache, odd length
        dict(name="prompt4", kind="prefill", chunks=1, new_lo=4095, new_hi=4095, cached_hi=0,
             hq=32, hkv=8, d=128, dtype="bfloat16", bits=4, block=16, window=0, sinks=0, layers=1,
             sizes=7),
        # a small decode batch of a float32 model with a window
        dict(name="window_f32", kind="decode", rows=8, lo=16, hi=2000, hq=14, hkv=2, d=64,
             dtype="float32", bits=32, block=16, window=256, sinks=4, layers=1, sizes=8),
        # long contexts of which a window and four sinks are read
        dict(name="window_decode", kind="decode", rows=64, lo=2048, hi=16384, hq=32, hkv=8, d=128,
             dtype="bfloat16", bits=16, block=16, window=1024, sinks=4, layers=2, sizes=9),
        # float32 chunks under a window
        dict(name="window_chunks_f32", kind="prefill", chunks=3, new_lo=100, new_hi=700,
             cached_hi=1500, hq=12, hkv=2, d=128, dtype="float32", bits=32, block=16, window=512,
             sinks=4, layers=1, sizes=10),
        # one long prompt under a window: the most arithmetic here
        dict(name="window_prompt", kind="prefill", chunks=1, new_lo=8191, new_hi=8191, cached_hi=0,
             hq=32, hkv=8, d=128, dtype="bfloat16", bits=16, block=16, window=1024, sinks=4,
             layers=1, sizes=11),
        # both: a decode step of long contexts over a 4-bit cache with a window, odd sizes
        dict(name="window4_step", kind="step", rows=97, lo=1000, hi=12000, hq=12, hkv=2, d=128,
             dtype="float16", bits=4, block=32, window=2047, sinks=13, layers=2, sizes=12),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("store", "append", "decode", "decode", "step", "step", "prefill", "prefill",
                       "prefill"))
    hq, hkv, d = rng.choice(HEADS)
    dtype = rng.choice(("float16", "bfloat16"))
    bits = 4 if kind in ("store", "append") else rng.choice((4, 4, 16, 16, 32))
    if bits == 32:
        dtype = "float32"
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, bits=bits, block=rng.choice((16, 32)),
                window=0, sinks=0, layers=1, sizes=rng.randrange(1 << 30))
    # 16- and 32-bit pools without a window are not among these operators
    if kind not in ("store", "append") and (bits != 4 or rng.random() < 0.4):
        case.update(window=_log(rng, 32, 4096), sinks=rng.choice((0, 1, 4, _log(rng, 1, 100))))
    if kind in ("store", "prefill"):
        lo = _log(rng, 16, 2048)
        case.update(new_lo=lo, new_hi=min(_log(rng, lo, 5000), 8 * lo),
                    cached_hi=0 if kind == "store" else rng.choice((0, _log(rng, 64, 4000))))
        case["chunks"] = max(1, min(rng.randint(1, 6), 8000 // case["new_hi"]))
        if bits == 32:  # the 32-bit matrix rate is a sixteenth of the 16-bit one
            case.update(chunks=min(3, case["chunks"]), new_lo=min(lo, 400),
                        new_hi=min(case["new_hi"], 900), cached_hi=min(case["cached_hi"], 1500))
    else:
        lo = _log(rng, 16, 4096)
        case.update(rows=_log(rng, 1, 96), lo=lo, hi=_log(rng, lo, 12288), layers=rng.randint(1, 2))
        if kind == "append":
            case["layers"] = 1
        # at most the tokens, and the bytes, of the longest listed decode
        while case["rows"] > 1 and (work(case)["bytes"] > 6e8 or
                                    sum(_lengths(case)[0]) * hkv * d > 290000 * 8 * 128):
            case["rows"] = case["rows"] * 3 // 4
    while work(case)["flops"] > 1.3e11:  # the largest listed prompt's
        case.update({k: case[k] * 3 // 4 for k in ("new_lo", "new_hi", "cached_hi")})
    return case


# ---- sizes: from the case alone ---------------------------------------------------------------

def _lengths(case):
    """Context lengths (cached + new) and new tokens of each sequence."""
    rng = random.Random(case["sizes"])
    if case["kind"] in ("store", "prefill"):
        new = [_log(rng, case["new_lo"], case["new_hi"]) for _ in range(case["chunks"])]
        return [n + rng.randint(0, case["cached_hi"]) for n in new], new
    return [_log(rng, case["lo"], case["hi"]) for _ in range(case["rows"])], [1] * case["rows"]


def _seen(case, p):
    """Keys that a query at position p sees."""
    w = case["window"]
    if not w or p < w:
        return p + 1
    return w + min(case["sinks"], p + 1 - w)


def _keys_read(case, n, m):
    """Keys of a context of n tokens that its last m queries see between them."""
    w = case["window"]
    first = n - m - w + 1 if w else 0  # the first query's window starts here
    return n if first <= 0 else n - first + min(case["sinks"], first)


def work(case):
    ctx, new = _lengths(case)
    hq, hkv, d, layers = case["hq"], case["hkv"], case["d"], case["layers"]
    size = 4 if case["dtype"] == "float32" else 2
    row4 = hkv * (d // 2 + d // 32)
    row = row4 if case["bits"] == 4 else hkv * d * size  # bytes of a cached K (or V) row
    tokens, pages = sum(new), sum(-(-n // case["block"]) for n in ctx)
    small = 4 * (pages + 2 * len(ctx) + 1)  # tables, lengths, offsets
    if case["kind"] == "store":  # 16-bit rows in and out, 4-bit rows written and read
        return {"bytes": 2 * tokens * (2 * hkv * d * size + 2 * row) + small, "flops": 0}
    tail = 2 * sum((n - 1) % case["block"] + 1 for n in ctx) * (row + hkv * d * size)
    if case["kind"] == "append":
        return {"bytes": 2 * tokens * (hkv * d * size + row) + tail + small, "flops": 0}
    keys = sum(_keys_read(case, n, m) for n, m in zip(ctx, new))
    pairs = sum(_seen(case, p) for n, m in zip(ctx, new) for p in range(n - m, n))
    moved = 2 * keys * row + 2 * tokens * hq * d * size
    if case["kind"] == "step":
        moved += 2 * tokens * (hkv * d * size + row) + tail
    return {"bytes": layers * moved + small, "flops": layers * 4 * hq * d * pairs}


# ---- inputs -----------------------------------------------------------------------------------

def _randn(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    return out.normal_(0.0, 1.0, generator=gen)


def _rows(gen, shape, dtype):
    """K or V rows as models have them: N(0, 1) with a few channels of larger values."""
    x = _randn(gen, shape, torch.float32)
    gain = torch.empty(shape[-2:], dtype=torch.float32, device=DEV).uniform_(generator=gen)
    return (x * torch.where(gain > 0.95, 4.0, 1.0)).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    ctx, new = _lengths(case)
    dt, bs, hkv, d, layers = (getattr(torch, case["dtype"]), case["block"], case["hkv"], case["d"],
                              case["layers"])
    gen, rng = torch.Generator(device=DEV).manual_seed(seed), random.Random(seed)
    pages = [-(-n // bs) for n in ctx]
    nb = sum(pages) + max(1, sum(pages) // 8)
    perm = list(range(nb))
    rng.shuffle(perm)
    rows, at, width = [], 0, max(pages)
    for p in pages:
        rows.append(perm[at:at + p] + [perm[at + p - 1]] * (width - p))
        at += p
    offs = [0]
    for n in new:
        offs.append(offs[-1] + n)
    s = dict(case=case, dt=dt, nb=nb, max_new=max(new), tables=_ints(rows), lens=_ints(ctx),
             offs=_ints(offs), q=[], k=[], v=[], k_new=[], v_new=[])
    if case["kind"] in ("append", "step"):  # the pages that the new tokens go to
        tails = [(n - 1) % bs + 1 for n in ctx]
        ends = [0]
        for n in tails:
            ends.append(ends[-1] + n)
        s.update(tail_tables=_ints([[r[p - 1]] for r, p in zip(rows, pages)]),
                 tail_lens=_ints(tails), tail_offs=_ints(ends), tail_total=ends[-1])
    elif case["kind"] == "store":
        s.update(tail_tables=s["tables"], tail_lens=s["lens"], tail_offs=_ints(
            [sum(ctx[:j]) for j in range(len(ctx) + 1)]), tail_total=sum(ctx))
    for _ in range(layers):
        if case["kind"] not in ("store", "append"):
            s["q"].append(_randn(gen, (offs[-1], case["hq"], d), dt))
        if case["kind"] in ("store", "append", "step"):
            s["k_new"].append(_rows(gen, (offs[-1], hkv, d), dt))
            s["v_new"].append(_rows(gen, (offs[-1], hkv, d), dt))
        for name in ("k", "v"):
            if case["bits"] != 4:
                s[name].append(_rows(gen, (nb, bs, hkv, d), dt))
            elif case["kind"] in ("store", "append"):  # pools as a cache allocates them
                s[name].append((torch.zeros((nb, hkv, bs, d // 2), dtype=torch.uint8, device=DEV),
                                torch.zeros((nb, hkv, bs, d // 32), dtype=torch.uint8, device=DEV)))
            else:
                s[name].append(_pack(_rows(gen, (nb, bs, hkv, d), dt).transpose(1, 2),
                                     case["dtype"]))
    return s


# ---- the definitions with elementary operations -------------------------------------------------

def _pack(x, dtype):
    """(codes uint8 [..., D/2], scales uint8 [..., D/32]) of rows [..., D]: per 32 values the
    smallest power of two 2^e with max|x| <= 7 * 2^e, and x / 2^e rounded to the nearest of
    0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code); the even dim in a byte's low half."""
    x = x.float().unflatten(-1, (-1, 32))
    frac, exp = torch.frexp(x.abs().amax(-1, keepdim=True))  # max = frac * 2^exp, frac in [.5, 1)
    e = (exp - 3 + (frac > 0.875).int()).clamp(E_LOW, E_HIGH[dtype])
    a = torch.ldexp(x.abs(), -e)
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int() + 8 * torch.signbit(x).int())
    code = code.flatten(-2)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), (e + 127)[..., 0].to(torch.uint8)


def _unpack(codes, scales):
    """float32 values of 4-bit rows."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    ex, half = (c >> 1) & 3, (c & 1).float()
    mag = torch.where(ex == 0, 0.5 * half, torch.ldexp(1.0 + 0.5 * half, ex - 1))
    mag = torch.where(c >= 8, -mag, mag).unflatten(-1, (-1, 32))
    return torch.ldexp(mag, (scales.int() - 127)[..., None]).flatten(-2)


def _paged_values(pool, tables, bits):
    """float32 rows [S, W * BS, Hkv, D] of the sequences' pages."""
    if bits == 4:
        rows = _unpack(pool[0][tables.long()], pool[1][tables.long()]).transpose(2, 3)
    else:
        rows = pool[tables.long()].float()
    return rows.flatten(1, 2)


def _store(pool, new, blocks, at, case):
    """New rows [T, Hkv, D] put at (block, offset) of a pool."""
    if case["bits"] == 4:
        codes, scales = _pack(new, case["dtype"])
        pool[0][blocks, :, at] = codes
        pool[1][blocks, :, at] = scales
    else:
        pool[blocks, at] = new


def _owners(offs, total):
    """Sequence of each of `total` rows, and its index within the sequence."""
    t = torch.arange(total, device=DEV, dtype=torch.int32)
    seq = torch.bucketize(t, offs[1:], right=True)
    return seq, t - offs[seq]


def _slots(s, total):
    """(block, offset) of the new rows: the last positions of their sequences."""
    bs = s["case"]["block"]
    seq, i = _owners(s["offs"], total)
    pos = s["lens"][seq] - (s["offs"][1:] - s["offs"][:-1])[seq] + i
    return s["tables"][seq, (pos // bs).long()].long(), (pos % bs).long()


def _held(s, layer):
    """The gathered rows of the pages that were written to."""
    seq, i = _owners(s["tail_offs"], s["tail_total"])
    return [_paged_values(s[n][layer], s["tail_tables"], s["case"]["bits"])[seq, i].to(s["dt"])
            for n in ("k", "v")]


def _attend(s, layer):
    """softmax(q k^T / sqrt(D)) v over the keys that each query sees, all sequences padded to
    the longest."""
    case, q = s["case"], s["q"][layer]
    hkv, d, g = case["hkv"], case["d"], case["hq"] // case["hkv"]
    total, rows = q.shape[0], s["max_new"]
    k = _paged_values(s["k"][layer], s["tables"], case["bits"]).transpose(1, 2)
    v = _paged_values(s["v"][layer], s["tables"], case["bits"]).transpose(1, 2)
    counts = s["offs"][1:] - s["offs"][:-1]
    i = torch.arange(rows, device=DEV, dtype=torch.int32)
    at = (s["offs"][:-1, None] + i).clamp(max=total - 1).long()                  # [S, rows]
    qs = q.float()[at].unflatten(2, (hkv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    pos = ((s["lens"] - counts)[:, None] + i)[:, :, None]                         # [S, rows, 1]
    key = torch.arange(k.shape[2], device=DEV, dtype=torch.int32)
    see = (key <= pos) & (key < s["lens"][:, None, None])
    if case["window"]:
        see &= (pos - key < case["window"]) | (key < case["sinks"])
    see = see.repeat_interleave(g, 1)[:, None]                                    # [S, 1, rows*g, keys]
    x = torch.matmul(qs, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    x = torch.where(see, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (rows, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)           # [S, rows, Hq, D]
    seq, j = _owners(s["offs"], total)
    return o[seq, j].to(q.dtype)


def _plain(s):
    case, outs = s["case"], []
    total = (s["q"] or s["k_new"])[0].shape[0]
    for layer in range(case["layers"]):
        if s["k_new"]:
            blocks, at = _slots(s, total)
            _store(s["k"][layer], s["k_new"][layer], blocks, at, case)
            _store(s["v"][layer], s["v_new"][layer], blocks, at, case)
        if s["q"]:
            outs.append(_attend(s, layer))
        if s["k_new"]:
            outs += _held(s, layer)
    return outs


# ---- the package's calls ----------------------------------------------------------------------

def _calls(s):
    from flexengine_amd import ops

    case, outs = s["case"], []
    kind, tables, lens, offs = case["kind"], s["tables"], s["lens"], s["offs"]
    seen = dict(window=case["window"], sinks=case["sinks"]) if case["window"] else {}
    for layer in range(case["layers"]):
        k, v = s["k"][layer], s["v"][layer]
        if case["bits"] == 4:
            k, v = ops.Kv4Pool(*k, s["dt"]), ops.Kv4Pool(*v, s["dt"])
        if kind == "store":
            ops.write_kv_ragged(s["k_new"][layer], s["v_new"][layer], k, v, tables, offs, lens)
        elif kind == "append":
            ops.write_kv_decode(s["k_new"][layer], s["v_new"][layer], k, v, tables, lens)
        elif kind == "decode":
            outs.append(ops.paged_decode(s["q"][layer], k, v, tables, lens, **seen))
        elif kind == "step":
            outs.append(ops.paged_decode(s["q"][layer], k, v, tables, lens, k_new=s["k_new"][layer],
                                         v_new=s["v_new"][layer], **seen))
        else:
            outs.append(ops.prefill_paged(s["q"][layer], k, v, tables, offs, lens, s["max_new"],
                                          **seen))
        if s["k_new"]:
            outs += ops.gather_kv(k, v, s["tail_tables"], s["tail_lens"], s["tail_offs"],
                                  s["tail_total"])
    return outs


def run(state):
    return _calls(state) if own else _plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------------------

def _nearest4(x, dtype):
    """The float64 values that rows [T, Hkv, D] have in 4 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], 32):
        b = x[..., c:c + 32].double()
        top = b.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, E_LOW)
        for t in range(E_LOW, E_HIGH[dtype]):  # one more while the largest does not fit
            e += (top > 7.0 * 2.0 ** t).double()
        a = b.abs() / 2.0 ** e
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        a = (torch.round(a / step) * step).clamp(max=6.0)
        out[..., c:c + 32] = torch.copysign(a * 2.0 ** e, b)
    return out


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_rows(s, name, layer, b, n):
    """float64 rows [n, Hkv, D] of a sequence, from its pages."""
    case, pool = s["case"], s[name][layer]
    blocks = s["tables"][b, :-(-n // case["block"])].long()
    if case["bits"] != 4:
        return pool[blocks].double().flatten(0, 1)[:n]
    codes = pool[0][blocks].transpose(1, 2).flatten(0, 1)[:n].long()
    table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=DEV)
    x = torch.empty(codes.shape[:2] + (case["d"],), dtype=torch.float64, device=DEV)
    x[..., 0::2] = table[codes % 16]
    x[..., 1::2] = table[codes // 16]
    scale = pool[1][blocks].transpose(1, 2).flatten(0, 1)[:n].double()
    return x * (2.0 ** (scale - 127.0)).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    hq, hkv, d, bs, outs = case["hq"], case["hkv"], case["d"], case["block"], []
    g = hq // hkv
    first = [sum(new[:b]) for b in range(len(new))]
    for layer in range(case["layers"]):
        out = torch.empty((sum(new), hq, d), dtype=torch.float64, device=DEV)
        held = {"k": [], "v": []}
        for b, (n, m) in enumerate(zip(ctx, new)):
            rows = {}
            for name in ("k", "v"):
                x = _exact_rows(s, name, layer, b, n)
                if s["k_new"]:
                    add = s[name + "_new"][layer][first[b]:first[b] + m]
                    x[n - m:] = _nearest4(add, case["dtype"]) if case["bits"] == 4 else add.double()
                    held[name].append(x if case["kind"] == "store" else x[(n - 1) // bs * bs:])
                rows[name] = x
            if not s["q"]:
                continue
            for at in range(0, m, 512):  # 512 queries at once
                end = min(at + 512, m)
                pos = torch.arange(n - m + at, n - m + end, device=DEV)[:, None]
                key = torch.arange(n, device=DEV)
                hide = key > pos
                if case["window"]:
                    hide |= (key <= pos - case["window"]) & (key >= case["sinks"])
                for h in range(hkv):
                    q = s["q"][layer][first[b] + at:first[b] + end, h * g:(h + 1) * g].double()
                    x = torch.matmul(q.transpose(0, 1), rows["k"][:, h].T.contiguous()) / math.sqrt(d)
                    p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
                    out[first[b] + at:first[b] + end, h * g:(h + 1) * g] = torch.matmul(
                        p, rows["v"][:, h].contiguous()).transpose(0, 1)
        if s["q"]:
            outs.append(out)
        if s["k_new"]:
            outs += [torch.cat(held["k"]), torch.cat(held["v"])]
    return outs
