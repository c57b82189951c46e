"""How the matrix-core attention over a paged cache divides its work, modelled on the CPU with the
constants of the emitted source: every partial within its area and on 128-byte lines of its own, every
workgroup in the grid, every arrival counter in its range, no index past 31 bits."""
import math
import random
import re

import numpy as np
import pytest

from sanic_amd import ir
from sanic_amd.program import Program

LINE_BYTES = 128


def emitted(T, NKV, REP, HD, BS, B, M, window=0, NB=100000):
    p = Program()
    q = p.input("q", (T, NKV * REP, HD), ir.BF16)
    kc, vc = (p.input(n, (NB, NKV, BS, HD), ir.BF16) for n in ("kc", "vc"))
    p.paged_attention("o", q, kc, vc, p.input("tables", (B, M), ir.U32), p.input("starts", (B + 1,), ir.U32), p.input("past", (B,), ir.U32),
                      window=window, out_dtype=ir.BF16)
    kind, source = p.emit(0)
    return kind, {m[1]: int(m[2]) for m in re.finditer(r"constexpr (?:int|long long) (\w+) = (-?\d+)(?:LL)?;", source)}


def key_tiles(c, past, new, tk):
    cut = lambda x: max(0, min(c["M"] * c["BS"], x))
    return max(1, -(-cut(past + new) // tk) - (cut(past + 1 - c["W"]) if c["W"] else 0) // tk)


def check(c, new, past):
    """The plan of requests with `new` rows each; returns (few-row parts, many-row parts)."""
    f32 = np.float32
    starts = [min(x, c["T"]) for x in np.concatenate(([0], np.cumsum(new)))]
    few, many = [], []
    for b, n in enumerate(np.diff(starts)):
        rows = int(n) * c["REP"]
        if rows == 0:
            continue
        if rows <= c["DR"]:
            few.append((b, rows, key_tiles(c, past[b], int(n), c["FEW_TK"])))
        else:
            many.append((b, rows, -(-rows // c["PR"]), key_tiles(c, past[b], int(n), c["MANY_TK"])))
    assert c["PITEMS"] or not many
    # few rows: equal runs of key tiles
    most = max([r for _, r, _ in few], default=0)
    unit = c.get("LINE", 1)
    stride = -(-most // unit) * unit
    groups = c["FEW_GROUPS"]
    if stride:
        groups = min(groups, c["DROWS"] // (2 * stride))
    assert groups >= 1
    run = max(f32(sum(k for _, _, k in few)) / f32(groups), f32(max([k for _, _, k in few], default=0)) / f32(c["MOST"]))
    run = int(max(1, math.ceil(run * f32(1.001))))
    at, top, spans = 0, -1, []          # spans: (request, first partial row, rows)
    for b, rows, k in few:
        w0, w1 = at // run, (at + k - 1) // run
        at, top = at + k, w1
        if w1 > w0:
            spans += [(b, w0 * 2 * stride + (s * 2 * stride if s else stride), rows) for s in range(w1 - w0 + 1)]
            assert (b + 1) * c["CPAD"] <= c["COUNTS"]
    parts_few = len(spans)
    for _, first, rows in spans:
        assert first + rows <= c["DROWS"]
    # many rows: tiles of PR rows, split over the keys
    tp, up = sum(t for _, _, t, _ in many), sum(t * k for _, _, t, k in many)
    part = 1 << 30
    if many and 2 * tp <= c["PSPLIT"]:
        room = c["PSPLIT"] - tp - 1
        part = int(min(1e9, max(1, math.ceil(up / room * 1.001)))) if room else int(1e9)
    items = tile = 0
    for b, rows, tiles, k in many:
        splits = min(-(-k // part), c["MOST"])
        if splits > 1:
            for t in range(tiles):
                n = min(c["PR"], rows - t * c["PR"])
                first = c["DROWS"] + (items + (tiles - 1 - t) * splits) * c["PR"]
                spans += [((b, t), first + s * c["PR"], n) for s in range(splits)]
                assert (c["B"] + tile + t + 1) * c["CPAD"] <= c["COUNTS"]
        items, tile = items + tiles * splits, tile + tiles
    for _, first, rows in spans:
        assert first + rows <= c["SLOTS"]
    # the lines of one request's (or tile's) partials are nobody else's: sums, then statistics
    for row in (c["HD"] * 4, 8):
        assert c["SLOTS"] * row % LINE_BYTES == 0
        owner = {}
        for who, first, rows in spans:
            for line in range(first * row // LINE_BYTES, ((first + rows) * row - 1) // LINE_BYTES + 1):
                assert owner.setdefault(line, who) == who, "a line of two requests' partials"
    rows = c["T"] * c["REP"]
    bound = rows // c["PR"] + min(c["B"], c["T"], rows // (c["DR"] + 1)) if rows > c["DR"] else 0
    grid = c["FEW_GROUPS"] + max(bound, c["PSPLIT"])
    assert items + top + 1 <= grid and (grid + 1) * run < 1 << 31
    return parts_few, len(spans) - parts_few


def test_decode_steps_share_no_line():
    """Heads of 64, four query heads a key head: a request's statistics are 32 bytes a part."""
    kind, c = emitted(64, 8, 4, 64, 16, 64, 256)
    assert kind == "operator:paged_attn[mfma]"
    few, many = check(c, [1] * 64, [37 * i % 4000 for i in range(64)])
    assert few > 64 and many == 0


def test_room_for_two_parts():
    """One tile of many rows where the partials have room for two parts alone."""
    _, c = emitted(40, 32, 1, 256, 16, 2, 256)
    check(c, [40, 0], [4000, 0])
    check(c, [39, 1], [4000, 4000])


def test_random_batches():
    r = random.Random(11)
    tried = parts = 0
    while tried < 150:
        B, NKV, REP, HD = int(2 ** r.uniform(0, 8)), r.choice([1, 2, 3, 4, 8, 16, 32]), r.choice([1, 2, 4, 7, 8, 16]), r.choice([16, 32, 48, 64, 80, 96, 128, 192, 256])
        BS, kind = r.choice([1, 8, 16, 24, 32, 64, 128]), r.choice(["one", "draft", "ragged", "mixed"])
        new = [{"one": lambda i: 1, "draft": lambda i: r.randint(0, 9), "ragged": lambda i: int(2 ** r.uniform(0, 9)),
                "mixed": lambda i: 1 if i else r.randint(1, 2000)}[kind](i) for i in range(B)]
        new[0] = max(new[0], 1)
        past = [int(2 ** r.uniform(0, 15)) for _ in range(B)]
        T = max(1, sum(new) + r.choice([0, 0, 5, -3]))
        M = max(-(-(a + n) // BS) for a, n in zip(past, new)) + 1
        kernel, c = emitted(T, NKV, REP, HD, BS, B, M, r.choice([0, 0, int(2 ** r.uniform(0, 13))]))
        if kernel != "operator:paged_attn[mfma]":
            continue
        parts += sum(check(c, new, past))
        tried += 1
    assert parts > 1000

@pytest.mark.parametrize("T,B,M,mfma", [(64, 64, 1 << 15, True), (1 << 16, 8192, 1 << 10, True), (1 << 22, 8192, 1 << 12, False)])
def test_runs_are_counted_in_31_bits(T, B, M, mfma):
    """A workgroup's first key tile is its number times the run's length: what could pass 31 bits takes
    the kernel without runs."""
    kind, c = emitted(T, 1, 16, 64, 64, B, M)
    assert (kind == "operator:paged_attn[mfma]") == mfma
