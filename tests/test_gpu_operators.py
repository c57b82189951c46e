"""The operators over ragged batches and paged caches on the GPU, through Program and
execute_static, against tests/paged_ref.py (f64 and whole numbers).

Tolerances count roundings: half a step of the stored type relative to the value
(`eps / 2`: bf16 2^-8, f16 2^-11, f32 2^-24), and for attention those of the kernel's f32 scores and
of its weights where they are rounded to the matrix cores' type; each is written at its test."""
import numpy as np
import pytest

import paged_ref as ref
from sanic_amd import ir
from sanic_amd.backend import decode, encode
from sanic_amd.program import NONE, OUTPUT, SCRATCH, STATE, Program

pytestmark = pytest.mark.gpu

HALF = {ir.F32: 2.0 ** -24, ir.BF16: 2.0 ** -8, ir.F16: 2.0 ** -11}


def stored(v, dtype):
    """The values a buffer of `dtype` holds after `v` was stored, f64."""
    v = np.asarray(v, np.float64)
    return decode(encode(v, dtype), dtype, v.size).reshape(v.shape)


def bind(dev, prog, vals, fill=0xA5):
    """A buffer for every one of the program's, inputs and states from `vals`, the rest bytes of `fill`."""
    out = {}
    for b in prog.buffers:
        if b.role == SCRATCH:
            continue
        if b.name in vals:
            out[b.name] = dev.from_values(vals[b.name], b.dtype)
        else:
            out[b.name] = dev.alloc(b.nbytes)
            out[b.name].upload(bytes([fill]) * b.nbytes)
    return out


def read(prog, bufs, name):
    b = prog.by_name[name]
    return bufs[name].read(b.dtype, int(np.prod(b.shape))).reshape(b.shape)


def words(prog, bufs, name):
    b = prog.by_name[name]
    return np.frombuffer(bufs[name].download(b.nbytes), np.uint32).reshape(b.shape).astype(np.int64)


FILL = int.from_bytes(b"\xa5" * 4, "little")


# ── block tables and slot maps ───────────────────────────────────────────────

def tables_program(B, F, M, T, block):
    p = Program()
    p.state("tables", (B, M), ir.U32)
    p.block_tables("plan", p.input("past", (B,), ir.U32), p.input("new", (B,), ir.U32), p.input("held", (B + 1,), ir.U32),
                   p.input("free", (F,), ir.U32), "tables", block=block, rows=T)
    return p


TABLES = {
    # name: (past, new, held or None = what past needs, free blocks, taken, M, block, rows or None)
    "one": ([0], [1], None, 4, 0, 2, 16, None),
    "one_in_its_block": ([5], [1], None, 4, 1, 2, 16, None),
    "fills_a_block": ([15, 16, 17], [1, 1, 1], None, 9, 0, 4, 16, None),
    "idle_ends_and_middle": ([3, 40, 0, 7, 9], [0, 5, 0, 1, 0], None, 9, 2, 9, 8, None),
    "nobody": ([3, 40], [0, 0], None, 3, 0, 9, 8, 7),
    "block_of_one": ([2, 0, 6], [3, 1, 2], None, 20, 0, 9, 1, None),
    "odd_block": ([24, 50, 23], [30, 1, 2], None, 20, 0, 9, 24, None),
    "held_more_than_needed": ([10, 33], [4, 1], [3, 4], 9, 0, 5, 16, None),
    "list_runs_out": ([0, 0, 16, 0], [40, 20, 1, 5], None, 4, 1, 9, 16, None),
    "list_is_used_up": ([0, 3], [4, 4], None, 3, 3, 9, 4, None),
    "taken_past_the_list": ([0, 3], [4, 4], None, 3, 7, 9, 4, None),
    "table_too_narrow": ([20, 0], [30, 9], None, 30, 0, 3, 8, None),
    "held_past_the_table": ([20, 9], [30, 9], [7, 2], 30, 0, 3, 8, None),
    "rows_cut": ([4, 5, 6], [10, 10, 10], None, 30, 0, 9, 8, 13),
    "rows_behind": ([4, 5, 6], [1, 0, 3], None, 30, 0, 9, 8, 300),
    "far_positions": ([(1 << 32) - 3], [2], [1], 30, 0, 3, 1 << 28, None),
}


@pytest.mark.parametrize("case", TABLES)
def test_block_tables(dev, case):
    past, new, held, F, taken, M, block, rows = TABLES[case]
    held = [min(-(-p // block), M) for p in past] if held is None else held
    check_tables(dev, past, new, held + [taken], F, M, block, sum(new) if rows is None else rows)


@pytest.mark.parametrize("B", [255, 256, 257, 1000, 8192])
def test_block_tables_many_requests(dev, B):
    g = np.random.default_rng(B)
    past = g.integers(0, 300, B)
    new = np.where(g.random(B) < 0.3, 0, g.integers(1, 40, B))
    block = 16
    held = -(-past // block) + (g.random(B) < 0.2)
    check_tables(dev, past, new, list(held) + [3], int(g.integers(B // 2, 3 * B)), 24, block, int(new.sum()) + 77)


def check_tables(dev, past, new, held, F, M, block, T):
    B = len(past)
    g = np.random.default_rng(7)
    ids = g.permutation(F + B * M)
    tables = np.full((B, M), NONE, np.int64)
    for b in range(B):
        n = min(int(held[b]), M)
        tables[b, :n] = ids[F + b * M:F + b * M + n]
    free = ids[:F]
    p = tables_program(B, F, M, T, block)
    bufs = bind(dev, p, {"past": past, "new": new, "held": held, "free": free, "tables": tables})
    exe = dev.prepare(p)
    starts, slots, positions, after, want = ref.block_tables(past, new, held, free, tables, block, T)
    n = starts[-1]
    for _ in range(2):   # the same call again writes the same
        exe.execute_static(bufs)
        assert words(p, bufs, "plan.starts").tolist() == starts
        assert words(p, bufs, "plan.held").tolist() == [int(x) for x in after]
        np.testing.assert_array_equal(words(p, bufs, "tables"), want)
        got = words(p, bufs, "plan.slots")
        assert got[:n].tolist() == slots and (got[n:] == FILL).all()
        got = words(p, bufs, "plan.positions")
        assert got[:n].tolist() == [x % (1 << 32) for x in positions] and (got[n:] == FILL).all()


# ── cache write ──────────────────────────────────────────────────────────────

def write_program(T, NKV, HD, NB, BS, B, src, dst, order="heads", fused=False):
    """order: the cache as [NB, NKV, BS, HD] or, read through a view, [NB, BS, NKV, HD]; fused: k
    and v are parts of one [T, 2·NKV·HD + 8] buffer."""
    p = Program()
    if fused:
        kv = p.input("kv", (T, 2 * NKV * HD + 8), src)
        part = lambda off: ir.reindex(kv, (T, NKV, HD), [(((1, 0),), 0), (((HD, 1), (1, 2)), off)])  # noqa: E731
        k, v = part(0), part(NKV * HD + 8)
    else:
        k, v = p.input("k", (T, NKV, HD), src), p.input("v", (T, NKV, HD), src)
    caches = []
    for n in ("kc", "vc"):
        if order == "heads":
            caches.append(p.state(n, (NB, NKV, BS, HD), dst))
        else:
            caches.append(ir.permute(p.state(n, (NB, BS, NKV, HD), dst), (0, 2, 1, 3)))
    p.cache_write("write", k, v, p.input("slots", (T,), ir.U32), p.input("starts", (B + 1,), ir.U32), *caches)
    return p


@pytest.mark.parametrize("T,NKV,HD,NB,BS,live,src,dst,order,fused", [
    (1, 1, 1, 1, 1, 1, ir.F32, ir.BF16, "heads", False),
    (1, 8, 64, 5, 16, 1, ir.F32, ir.BF16, "heads", False),
    (9, 3, 24, 4, 5, 7, ir.F32, ir.F16, "heads", False),
    (40, 2, 80, 9, 16, 33, ir.BF16, ir.BF16, "heads", False),
    (40, 2, 7, 9, 16, 40, ir.F16, ir.F32, "heads", False),
    (70, 4, 128, 11, 24, 64, ir.F16, ir.F16, "tokens", False),
    (33, 4, 64, 11, 8, 30, ir.F32, ir.BF16, "tokens", True),
    (33, 4, 12, 11, 8, 33, ir.BF16, ir.F32, "heads", True),
    (600, 8, 128, 70, 16, 0, ir.BF16, ir.BF16, "heads", False),
    (600, 8, 128, 70, 16, 599, ir.BF16, ir.BF16, "heads", False),
])
def test_cache_write(dev, T, NKV, HD, NB, BS, live, src, dst, order, fused):
    g = np.random.default_rng(T * HD)
    B = 3
    p = write_program(T, NKV, HD, NB, BS, B, src, dst, order, fused)
    slots = g.permutation(NB * BS)[:T] if T <= NB * BS else g.integers(0, NB * BS, T)
    if T > 3:
        # no slot, and slots behind the pool
        slots[[0, 2]] = NONE, NB * BS
    # values at the edges of the types beside ordinary ones
    k, v = (g.standard_normal((T, NKV, HD)) * np.exp2(g.integers(-20, 10, (T, 1, 1))) for _ in range(2))
    k[0, 0, 0] = 65504.0
    vals = {"slots": slots, "starts": [0, live // 2, live // 2, live]}
    if fused:
        vals["kv"] = np.concatenate((k.reshape(T, -1), np.full((T, 8), 7.0), v.reshape(T, -1)), 1)
    else:
        vals.update(k=k, v=v)
    old = {n: g.standard_normal(p.by_name[n].shape) for n in ("kc", "vc")}
    bufs = bind(dev, p, {**vals, **old})
    dev.prepare(p).execute_static(bufs)
    for name, rows in (("kc", k), ("vc", v)):
        want = stored(old[name], dst)
        flat = want if order == "tokens" else want.transpose(0, 2, 1, 3).copy()
        flat = flat.reshape(NB * BS, NKV, HD)
        with np.errstate(over="ignore"):
            for r in range(live):
                if slots[r] < NB * BS:
                    flat[slots[r]] = stored(stored(rows[r], src), dst)
        want = flat.reshape(NB, BS, NKV, HD)
        np.testing.assert_array_equal(read(p, bufs, name), want if order == "tokens" else want.transpose(0, 2, 1, 3))


def test_cache_write_keeps_what_is_not_finite(dev):
    p = write_program(4, 1, 8, 2, 4, 1, ir.F32, ir.BF16)
    k = np.zeros((4, 1, 8))
    k[0], k[1], k[2] = np.inf, -np.inf, np.nan
    bufs = bind(dev, p, {"k": k, "v": k, "slots": [3, 1, 0, 6], "starts": [0, 4], "kc": np.ones((2, 1, 4, 8)), "vc": np.ones((2, 1, 4, 8))})
    dev.prepare(p).execute_static(bufs)
    for name in ("kc", "vc"):
        got = read(p, bufs, name)
        assert (got[0, 0, 3] == np.inf).all() and (got[0, 0, 1] == -np.inf).all() and np.isnan(got[0, 0, 0]).all()
        assert (got[1, 0, 2] == 0).all() and (got[0, 0, 2] == 1).all() and (got[1, 0, [0, 1, 3]] == 1).all()


# ── attention ────────────────────────────────────────────────────────────────

def attn_program(T, NH, NKV, HD, NB, BS, B, M, dq, dc, do, window, scale=None, order="heads", q_order="tokens"):
    p = Program()
    q = p.input("q", (T, NH, HD), dq) if q_order == "tokens" else ir.permute(p.input("q", (NH, T, HD), dq), (1, 0, 2))
    c = []
    for n in ("kc", "vc"):
        c.append(p.input(n, (NB, NKV, BS, HD), dc) if order == "heads" else
                 ir.permute(p.input(n, (NB, BS, NKV, HD), dc), (0, 2, 1, 3)))
    p.paged_attention("o", q, *c, p.input("tables", (B, M), ir.U32), p.input("starts", (B + 1,), ir.U32), p.input("past", (B,), ir.U32),
                      scale=scale, window=window, out_dtype=do)
    return p


class Batch:
    """A ragged batch over a pool whose unused places hold NaN."""

    def __init__(self, past, new, NKV, rep, HD, BS, dq=ir.BF16, dc=None, do=None, window=0, pad=0, spread=1.0, spare=2, scale=None, seed=0):
        g = np.random.default_rng(seed * 7919 + sum(past) + 31 * sum(new) + HD)
        dc, do = dq if dc is None else dc, dq if do is None else do
        self.past, self.new, self.window, self.types = past, new, window, (dq, dc, do)
        self.scale = scale
        self.B, self.T = len(past), max(1, sum(new) + pad)
        self.NKV, self.rep, self.HD, self.BS = NKV, rep, HD, BS
        have = [-(-(a + b) // BS) for a, b in zip(past, new)]
        self.M = max(max(have), 1) + 1
        self.NB = sum(have) + spare
        ids = g.permutation(self.NB)
        self.tables = np.full((self.B, self.M), NONE, np.int64)
        at = 0
        kc = np.full((self.NB, NKV, BS, HD), np.nan)
        vc = kc.copy()
        for b, n in enumerate(have):
            self.tables[b, :n] = ids[at:at + n]
            at += n
            for i in range(n):
                w = min(BS, past[b] + new[b] - i * BS)
                kc[self.tables[b, i], :, :w] = g.standard_normal((NKV, w, HD)) * spread
                vc[self.tables[b, i], :, :w] = g.standard_normal((NKV, w, HD))
        self.starts = np.concatenate(([0], np.cumsum(new)))
        self.q = stored(g.standard_normal((self.T, NKV * rep, HD)), dq)
        self.kc, self.vc = stored(kc, dc), stored(vc, dc)

    def program(self, **kw):
        return attn_program(self.T, self.NKV * self.rep, self.NKV, self.HD, self.NB, self.BS, self.B, self.M, *self.types, self.window,
                            self.scale, **kw)

    def values(self):
        return {"q": self.q, "kc": self.kc, "vc": self.vc, "tables": self.tables, "starts": self.starts, "past": self.past}

    def want(self):
        return ref.paged_attention(self.q, self.kc, self.vc, self.tables, self.starts, self.past,
                                   1.0 / np.sqrt(self.HD) if self.scale is None else self.scale, self.window)

    def check(self, got, kind):
        o, mag = self.want()
        n = min(int(self.starts[-1]), self.T)
        got, o, mag = got[:n], o[:n], mag[:n]
        dq, dc, do = self.types
        # the scores in f32: each of the HD products and sums by half a step of 24 bits, so a weight is
        # off by a factor of at most 1 + HD·2^-24·Σ|q·k|·scale and an output, a quotient of two such
        # sums, by twice that of the values' mean; |q·k| sums stay under 4·HD for these inputs at
        # spread 1, and the exponential adds 2^-20. Weights rounded to bf16 or f16 add half a step of
        # theirs to the products and to their sum.
        f32 = 2.0 * (self.HD * 2.0 ** -24 * 4 * self.HD / np.sqrt(self.HD) + 2.0 ** -20)
        weights = 0.0 if "plain" in kind else 2.0 * HALF[dc]
        tol = HALF[do] * np.abs(o) + (1 + HALF[do]) * (f32 + weights) * mag + 1e-30
        worst = np.abs(got - o) / tol
        assert not np.isnan(got).any(), np.argwhere(np.isnan(got))[:5].tolist()
        assert (worst <= 1).all(), (kind, float(worst.max()), np.argwhere(worst > 1)[:5])

    def run(self, dev, **kw):
        p = self.program(**kw)
        vals = self.values()
        if kw.get("order") == "tokens":
            vals["kc"], vals["vc"] = vals["kc"].transpose(0, 2, 1, 3), vals["vc"].transpose(0, 2, 1, 3)
        if kw.get("q_order") == "heads":
            vals["q"] = vals["q"].transpose(1, 0, 2)
        bufs = bind(dev, p, vals)
        exe = dev.prepare(p)
        exe.execute_static(bufs)
        first = bufs["o"].download()
        exe.execute_static(bufs)
        assert bufs["o"].download() == first, "two runs differ"
        n = int(self.starts[-1]) * self.NKV * self.rep * self.HD * ir.dtype_bytes(self.types[2], 1)
        assert first[n:] == b"\xa5" * (len(first) - n), "rows behind the last request were written"
        self.check(read(p, bufs, "o"), exe.stage_kernel(0))
        return exe.stage_kernel(0)


ATTN = {
    "first_token": dict(past=[0], new=[1], NKV=1, rep=1, HD=64, BS=16),
    "second_token": dict(past=[1], new=[1], NKV=2, rep=4, HD=64, BS=16),
    "decode": dict(past=[100, 0, 15, 16, 31, 700], new=[1] * 6, NKV=2, rep=4, HD=64, BS=16),
    "decode_128": dict(past=[100, 63, 64, 1000], new=[1] * 4, NKV=2, rep=4, HD=128, BS=16),
    "decode_f16": dict(past=[100, 63, 2500], new=[1] * 3, NKV=2, rep=8, HD=128, BS=32, dq=ir.F16),
    "decode_one_head": dict(past=[333], new=[1], NKV=1, rep=1, HD=128, BS=64),
    "decode_many_heads_a_key": dict(past=[333, 20], new=[1, 1], NKV=1, rep=32, HD=64, BS=16),
    "decode_heads_of_their_own": dict(past=[333, 20], new=[1, 1], NKV=12, rep=1, HD=64, BS=16),
    "decode_seven_heads": dict(past=[333, 20], new=[1, 1], NKV=2, rep=7, HD=64, BS=16),
    "drafts": dict(past=[100, 7, 0, 300], new=[5, 5, 5, 3], NKV=2, rep=4, HD=64, BS=16),
    "drafts_33_rows": dict(past=[100, 90], new=[11, 11], NKV=2, rep=3, HD=64, BS=16),
    "prompt": dict(past=[0], new=[200], NKV=2, rep=4, HD=64, BS=16),
    "prompt_128": dict(past=[0, 0], new=[129, 65], NKV=2, rep=2, HD=128, BS=64),
    "chunk": dict(past=[130, 63], new=[70, 64], NKV=2, rep=4, HD=64, BS=32),
    "chunk_f16": dict(past=[130], new=[90], NKV=1, rep=4, HD=128, BS=16, dq=ir.F16),
    "mixed": dict(past=[500, 40, 9, 0, 77], new=[1, 150, 0, 33, 1], NKV=2, rep=4, HD=64, BS=16, pad=9),
    "idle_ends": dict(past=[50, 40, 9], new=[0, 3, 0], NKV=1, rep=4, HD=64, BS=16, pad=3),
    "nobody": dict(past=[50, 40], new=[0, 0], NKV=1, rep=4, HD=64, BS=16, pad=3),
    "window_decode": dict(past=[500, 40, 63], new=[1, 1, 1], NKV=2, rep=4, HD=64, BS=16, window=64),
    "window_of_one": dict(past=[500, 40], new=[1, 3], NKV=2, rep=4, HD=64, BS=16, window=1),
    "window_chunk": dict(past=[300, 0], new=[120, 130], NKV=1, rep=4, HD=64, BS=16, window=50),
    "window_128": dict(past=[300, 0], new=[70, 130], NKV=1, rep=4, HD=128, BS=16, window=100),
    "block_of_one": dict(past=[90], new=[3], NKV=1, rep=4, HD=64, BS=1),
    "block_24": dict(past=[190, 23, 24], new=[1, 30, 1], NKV=1, rep=4, HD=64, BS=24),
    "block_128": dict(past=[190, 127, 128], new=[1, 30, 1], NKV=1, rep=4, HD=64, BS=128),
    "block_100": dict(past=[190, 99], new=[1, 30], NKV=1, rep=4, HD=128, BS=100),
    "head_32": dict(past=[190, 99], new=[1, 30], NKV=2, rep=4, HD=32, BS=16),
    "head_48": dict(past=[190, 99], new=[1, 30], NKV=2, rep=4, HD=48, BS=16),
    "head_80": dict(past=[190, 99], new=[1, 30], NKV=2, rep=4, HD=80, BS=16),
    "head_96": dict(past=[190, 99], new=[1, 30], NKV=2, rep=2, HD=96, BS=16),
    "head_112": dict(past=[190, 99], new=[1, 30], NKV=2, rep=2, HD=112, BS=16),
    "head_160": dict(past=[190, 99], new=[1, 30], NKV=1, rep=2, HD=160, BS=16),
    "head_256": dict(past=[190, 99], new=[1, 30], NKV=1, rep=2, HD=256, BS=16),
    "head_7": dict(past=[190, 9], new=[1, 30], NKV=2, rep=2, HD=7, BS=16),
    "head_1": dict(past=[190, 9], new=[1, 30], NKV=2, rep=2, HD=1, BS=16),
    "head_500": dict(past=[90, 9], new=[1, 10], NKV=1, rep=2, HD=500, BS=16),
    "f32": dict(past=[190, 9], new=[1, 30], NKV=2, rep=2, HD=64, BS=16, dq=ir.F32),
    "f32_cache_bf16": dict(past=[190, 9], new=[1, 30], NKV=2, rep=2, HD=64, BS=16, dq=ir.F32, dc=ir.BF16),
    "bf16_out_f32": dict(past=[190, 9, 30], new=[1, 30, 5], NKV=2, rep=2, HD=64, BS=16, do=ir.F32),
    "bf16_cache_f16": dict(past=[190, 9], new=[1, 30], NKV=2, rep=2, HD=64, BS=16, dc=ir.F16),
    "scale": dict(past=[190, 9, 40], new=[1, 30, 4], NKV=2, rep=2, HD=64, BS=16, scale=0.02),
    "many_short": dict(past=[3 * i % 41 for i in range(90)], new=[1 + (i % 7 == 0) for i in range(90)], NKV=2, rep=4, HD=64, BS=16),
    "long_and_short": dict(past=[9000] + [30] * 9, new=[1] * 10, NKV=1, rep=4, HD=64, BS=16),
    "long_chunk": dict(past=[3000], new=[40], NKV=1, rep=4, HD=64, BS=16),
    "room_for_two_parts": dict(past=[100], new=[40], NKV=32, rep=1, HD=256, BS=16),
    "long_drafts_128": dict(past=[4000, 10], new=[4, 4], NKV=1, rep=8, HD=128, BS=16),
}


@pytest.mark.parametrize("case", ATTN)
def test_paged_attention(dev, case):
    print(case, Batch(**ATTN[case]).run(dev))


@pytest.mark.parametrize("order,q_order", [("tokens", "tokens"), ("heads", "heads"), ("tokens", "heads")])
@pytest.mark.parametrize("HD", [64, 128, 20])
def test_paged_attention_orders(dev, order, q_order, HD):
    Batch(past=[70, 200, 4], new=[40, 1, 3], NKV=2, rep=4, HD=HD, BS=16).run(dev, order=order, q_order=q_order)


def _with_bad_pages(dtype, HD, new):
    t = Batch(past=[200, 64, 30], new=[new, new, new], NKV=2, rep=4, HD=HD, BS=16, dq=dtype, pad=2)
    # no block, a block behind the pool, and a request that has lost all of its blocks
    t.tables[0, 3], t.tables[0, 7], t.tables[1, 0] = NONE, t.NB, t.NB + 5
    t.tables[2, :] = NONE
    return t


@pytest.mark.parametrize("dtype,HD,new", [(ir.BF16, 64, 1), (ir.BF16, 128, 5), (ir.F16, 64, 60), (ir.F32, 24, 3)])
def test_paged_attention_without_blocks(dev, dtype, HD, new):
    t = _with_bad_pages(dtype, HD, new)
    t.run(dev)
    assert (t.want()[0][t.starts[2]:t.starts[3]] == 0).all()


def test_paged_attention_starts_behind_the_rows(dev):
    """Starts past T are T: the rows that exist are answered, nothing else is touched."""
    t = Batch(past=[30, 40], new=[3, 50], NKV=1, rep=4, HD=64, BS=16)
    t.T = 20
    t.q = t.q[:20]
    p = t.program()
    bufs = bind(dev, p, {**t.values(), "starts": [0, 3, 1 << 31]})
    exe = dev.prepare(p)
    exe.execute_static(bufs)
    t.check(read(p, bufs, "o"), exe.stage_kernel(0))


@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_positions_behind_the_table(dev, new):
    """A past beyond the table sees the table's keys (here every place of every block is written)."""
    t = Batch(past=[64 - new], new=[new], NKV=1, rep=4, HD=64, BS=16)
    t.past = [(1 << 32) - 1 - new]
    t.window = 0
    t.tables[:, -1] = NONE
    t.run(dev)


@pytest.mark.parametrize("dtype,new", [(ir.BF16, 1), (ir.BF16, 40), (ir.F16, 5), (ir.F32, 3)])
def test_paged_attention_large_scores(dev, dtype, new):
    """Scores of some thousands: one key takes all the weight, and nothing overflows."""
    t = Batch(past=[150], new=[new], NKV=1, rep=4, HD=64, BS=16, dq=dtype, spread=300.0)
    o, _ = t.want()
    p = t.program()
    bufs = bind(dev, p, t.values())
    exe = dev.prepare(p)
    exe.execute_static(bufs)
    got = read(p, bufs, "o")
    assert np.isfinite(got).all()
    # the two largest scores of a row as a rule lie far apart; a row is compared where they differ by
    # more than 40, so that every other weight is below e^-40
    s = np.einsum("rhd,kd->rhk", t.q, t.kc[t.tables[0, np.arange(150 + new) // 16].astype(int), 0, np.arange(150 + new) % 16]) / 8.0
    for r in range(new):
        s[r, :, 151 + r:] = -np.inf
    top = np.sort(s, -1)
    sure = top[..., -1] - top[..., -2] > 40
    assert sure.any()
    assert (np.abs(got - o)[sure] <= HALF[t.types[2]] * np.abs(o)[sure] + 1e-12).all()


@pytest.mark.parametrize("new", [1, 40])
def test_paged_attention_nan_in_sight(dev, new):
    """A NaN among a row's own keys is in its output, and in no other request's."""
    t = Batch(past=[150, 20], new=[new, new], NKV=1, rep=2, HD=64, BS=16)
    t.kc[t.tables[0, 2], 0, 5, 3] = np.nan
    p = t.program()
    bufs = bind(dev, p, t.values())
    dev.prepare(p).execute_static(bufs)
    got = read(p, bufs, "o")
    assert np.isnan(got[:new]).all() and np.isfinite(got[new:]).all()


@pytest.mark.parametrize("dtype", [ir.BF16, ir.F16])
@pytest.mark.parametrize("HD", [64, 128, 80])
@pytest.mark.parametrize("new,at", [(6, 4), (6, 0), (90, 61), (200, 130)])
def test_paged_attention_not_finite_behind_some_rows(dev, dtype, HD, new, at):
    """What is not finite at one of the step's own tokens reaches the rows from there on, and no
    element of the rows before it (0 · NaN would, were the masked keys multiplied)."""
    for value in (np.nan, np.inf, -np.inf):
        t = Batch(past=[70], new=[new], NKV=2, rep=3, HD=HD, BS=16, dq=dtype)
        where = (int(t.tables[0, (70 + at) // 16]), slice(None), (70 + at) % 16)
        t.vc[where + (5,)] = value
        t.kc[where + (3,)] = np.nan if at % 2 else 1.0     # a key too: its score is NaN where it is seen
        p = t.program()
        bufs = bind(dev, p, t.values())
        exe = dev.prepare(p)
        exe.execute_static(bufs)
        got = read(p, bufs, "o")
        clean = Batch(past=[70], new=[new], NKV=2, rep=3, HD=HD, BS=16, dq=dtype)
        clean.starts = np.array([0, at])
        clean.check(got, exe.stage_kernel(0))
        late = got[at:]
        if at % 2:
            assert np.isnan(late).all()
        else:
            assert np.isfinite(np.delete(late, 5, axis=2)).all()
            assert np.isnan(late[..., 5]).all() if np.isnan(value) else (late[..., 5] == value).all()


# ── verification of drafts ───────────────────────────────────────────────────

def verify_program(T, B, V, dp, dq):
    p = Program()
    p.verify_drafts("check", p.input("p", (T, V), dp), None if dq is None else p.input("q", (T, V), dq), p.input("tokens", (T,), ir.U32),
                    p.input("starts", (B + 1,), ir.U32), p.input("u", (T,), ir.F32), p.input("draw", (B,), ir.F32))
    return p


def check_verify(dev, vals, dp, dq):
    T, V = vals["p"].shape
    B = len(vals["draw"])
    prog = verify_program(T, B, V, dp, dq)
    vals = dict(vals, p=stored(vals["p"], dp), u=stored(vals["u"], ir.F32), draw=stored(vals["draw"], ir.F32))
    if dq is not None:
        vals["q"] = stored(vals["q"], dq)
    bufs = bind(dev, prog, vals)
    exe = dev.prepare(prog)
    want, accepted = ref.verify(vals["p"], vals.get("q") if dq is not None else None, vals["tokens"], vals["starts"], vals["u"], vals["draw"])
    for _ in range(3):
        exe.execute_static(bufs)
        got = words(prog, bufs, "check.tokens")
        assert words(prog, bufs, "check.accepted").tolist() == accepted
        assert got[:len(want)].tolist() == want and (got[len(want):] == FILL).all()
    return want, accepted


def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 2048, 2049, 32003, 128256])
@pytest.mark.parametrize("dp,dq", [(ir.F32, ir.F32), (ir.BF16, ir.BF16), (ir.F16, ir.F32), (ir.F32, None), (ir.BF16, None)])
def test_verify_drafts(dev, V, dp, dq):
    g = np.random.default_rng(V)
    counts = [5, 1, 0, 9, 3, 2]
    T, B = sum(counts) + 4, len(counts)
    logits = g.standard_normal((T, V)) * 2
    vals = {"p": _softmax(logits), "q": _softmax(logits + 0.5 * g.standard_normal((T, V))),
            "tokens": np.array([g.choice(V, p=_softmax(l)) for l in logits]), "starts": np.concatenate(([0], np.cumsum(counts))),
            "u": g.random(T), "draw": g.random(B)}
    want, accepted = check_verify(dev, vals, dp, dq)
    assert len(want) == sum(counts)


def test_verify_all_and_none_accepted(dev):
    g = np.random.default_rng(3)
    V, T = 500, 12
    p = _softmax(g.standard_normal((T, V)))
    vals = {"p": p, "q": p, "tokens": g.integers(0, V, T), "starts": [0, 6, 12], "u": np.zeros(T), "draw": [0.0, 0.999]}
    assert check_verify(dev, vals, ir.F32, ir.F32)[1] == [5, 5]
    # q far above p at every draft: refused at once; u = 1 refuses p == q and leaves no difference: drawn from p
    q = p.copy()
    q[np.arange(T - 1), vals["tokens"][1:]] = 1.0
    assert check_verify(dev, dict(vals, q=q, u=np.full(T, 0.99)), ir.F32, ir.F32)[1] == [0, 0]
    assert check_verify(dev, dict(vals, u=np.ones(T)), ir.F32, ir.F32)[1] == [0, 0]


def test_verify_nothing_left_over_a_large_vocabulary(dev):
    """Refused with p == q: the token is drawn from p, also where many workgroups share the row."""
    g = np.random.default_rng(8)
    V, T = 50021, 4
    p = stored(_softmax(g.standard_normal((T, V))), ir.F32)
    vals = {"p": p, "q": p, "tokens": g.integers(0, V, T), "starts": [0, 2, 4], "u": np.ones(T), "draw": [0.37, 0.81]}
    assert check_verify(dev, vals, ir.F32, ir.F32)[1] == [0, 0]


@pytest.mark.parametrize("drafts", [63, 64, 65, 130])
def test_verify_many_drafts(dev, drafts):
    g = np.random.default_rng(drafts)
    V, T = 40, 2 * (drafts + 1)
    p = _softmax(g.standard_normal((T, V)))
    vals = {"p": p, "q": p, "tokens": g.integers(0, V, T), "starts": [0, drafts + 1, T], "u": np.full(T, 0.5), "draw": [0.3, 0.6]}
    vals["u"][drafts + 1 + drafts - 2] = 1.0     # the second request's last draft but one is refused
    assert check_verify(dev, vals, ir.F32, ir.F32)[1] == [drafts, drafts - 2]


def test_verify_odd_inputs(dev):
    """Tokens outside the vocabulary and NaN are refused, weights that are not positive count as 0,
    and a row without weight gives no token."""
    g = np.random.default_rng(5)
    V = 300
    p = _softmax(g.standard_normal((12, V)))
    vals = {"p": p.copy(), "q": p.copy(), "tokens": g.integers(0, V, 12), "starts": [0, 3, 6, 9, 12], "u": np.full(12, 0.1), "draw": [0.5, 1.0, 0.2, 0.7]}
    vals["tokens"][1] = V
    vals["tokens"][4] = NONE
    vals["p"][6] = 0.0
    vals["q"][6] = 0.0
    vals["p"][9, vals["tokens"][10]] = np.nan
    vals["p"][9, 7] = -1.0
    for dq in (ir.F32, None):
        want, accepted = check_verify(dev, vals, ir.F32, dq)
        assert accepted[:2] == [0, 0] and want[6] == NONE


def test_verify_starts_behind_the_rows(dev):
    g = np.random.default_rng(6)
    V, T = 300, 7
    p = _softmax(g.standard_normal((T, V)))
    check_verify(dev, {"p": p, "q": p, "tokens": g.integers(0, V, T), "starts": [0, 4, 1 << 30, 1 << 31], "u": np.full(T, 0.1),
                       "draw": [0.5, 0.1, 0.2]}, ir.F32, ir.F32)
