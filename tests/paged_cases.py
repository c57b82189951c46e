"""Batches whose values are not finite, with what the definition gives for them."""
import numpy as np

from sanic_amd import ir
from sanic_amd.program import NONE
from test_gpu_operators import Batch, stored, tables_program


class OddValue:
    """One value of a key that stands in a tile every row sees whole, and its effect: a value that is
    not finite reaches that dim of every row that sees its key, whatever the key's weight, and nothing
    else."""

    def __init__(self, value, at, far=False, HD=64, past=200, new=1, dim=5, dq=ir.BF16, do=None, rep=4, NKV=2):
        kw = dict(past=[past, 40], new=[new, new], NKV=NKV, rep=rep, HD=HD, BS=16, dq=dq, do=do)
        self.batch, self.clean = Batch(**kw), Batch(**kw)
        where = (int(self.batch.tables[0, at // 16]), slice(None), at % 16)
        if far:       # a score so far below the others that the weight is 0 in 32 bits
            for t in (self.batch, self.clean):
                t.q[:, :, 0] = 8.0
                t.kc[where + (0,)] = stored(-400.0, dq)
        self.clean.vc[where + (dim,)] = 0.0
        self.batch.vc[where + (dim,)] = value
        self.value, self.dim, self.at = value, dim, at

    def check(self, got, kind):
        t = self.batch
        rows = slice(0, t.new[0])
        seen = got[rows][..., self.dim]
        assert np.isnan(seen).all() if np.isnan(self.value) else (seen == self.value).all(), seen.ravel()[:8]
        got = got.copy()
        got[rows][..., self.dim] = self.clean.want()[0][rows][..., self.dim]
        self.clean.check(got, kind)


ODD_VALUES = {
    f"{n}_{np.format_float_positional(v, trim='-')}{'_far' if far else ''}": dict(kw, value=v, far=far)
    for n, kw in {
        "token": dict(at=70), "token_128": dict(at=70, HD=128), "token_f16": dict(at=70, dq=ir.F16), "drafts": dict(at=33, new=5), "drafts_80": dict(at=33, new=5, HD=80),
        "token_f32_out": dict(at=70, do=ir.F32), "chunk": dict(at=70, new=60), "chunk_128": dict(at=70, new=40, HD=128), "chunk_f32_out": dict(at=70, new=60, do=ir.F32),
        "chunk_f16": dict(at=70, new=60, dq=ir.F16), "head_24": dict(at=70, HD=24), "first_key": dict(at=0, new=40), "split": dict(at=600, past=4000, rep=2, NKV=1),
    }.items() for v in (np.inf, -np.inf, np.nan) for far in (False, True)}


class OddKey:
    """One key with an element of −inf against queries that are positive there: a score of −inf, so a
    weight of 0, and every row is as if the key were not there. The others see their own keys."""

    def __init__(self, HD, dim, new=1, at=70, dq=ir.BF16, value=-np.inf):
        kw = dict(past=[200, 40], new=[new, new], NKV=2, rep=4, HD=HD, BS=16, dq=dq)
        self.batch, self.clean = Batch(**kw), Batch(**kw)
        where = (int(self.batch.tables[0, at // 16]), slice(None), at % 16)
        for t in (self.batch, self.clean):
            t.q[:, :, dim] = np.abs(t.q[:, :, dim]) + 0.5
            t.q[:] = stored(t.q, dq)
        self.batch.kc[where + (dim,)] = value
        # so far below the others that its weight is 0 in 64 bits too
        self.clean.kc[where + (dim,)] = stored(-60000.0, dq)

    def check(self, got, kind):
        assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:4]
        self.clean.check(got, kind)


ODD_KEYS = {f"head_{HD}_dim_{dim}_rows_{new}_{'f16' if dq == ir.F16 else 'bf16'}": dict(HD=HD, dim=dim, new=new, dq=dq)
            for HD, dim in ((16, 15), (48, 40), (80, 72), (112, 111), (144, 137), (208, 207), (64, 63), (24, 23)) for new in (1, 5, 50)
            for dq in ((ir.BF16, ir.F16) if HD == 80 else (ir.BF16,))}


class OddQuery:
    """A NaN in a query row makes the row NaN, and no other."""

    def __init__(self, past, new, row, HD=64, NKV=2, rep=4, dq=ir.BF16, do=None):
        self.batch = Batch(past=past, new=new, NKV=NKV, rep=rep, HD=HD, BS=16, dq=dq, do=do)
        self.clean = Batch(past=past, new=new, NKV=NKV, rep=rep, HD=HD, BS=16, dq=dq, do=do)
        self.row, self.head = row, NKV * rep - 1
        self.batch.q[row, self.head, 3] = np.nan

    def check(self, got, kind):
        assert np.isnan(got[self.row, self.head]).all(), got[self.row, self.head][:8]
        got = got.copy()
        got[self.row, self.head] = self.clean.want()[0][self.row, self.head]
        self.clean.check(got, kind)


ODD_QUERIES = {
    "first_token": dict(past=[0], new=[1], row=0), "token": dict(past=[70, 9], new=[1, 1], row=0), "token_split": dict(past=[4000, 9], new=[1, 1], row=0, NKV=1, rep=2),
    "draft": dict(past=[70, 9], new=[5, 5], row=7), "draft_128": dict(past=[700, 9], new=[5, 5], row=3, HD=128), "draft_f32_out": dict(past=[70, 9], new=[5, 5], row=2, do=ir.F32),
    "chunk": dict(past=[70, 9], new=[50, 5], row=13), "chunk_split": dict(past=[3000], new=[40], row=39, NKV=1), "head_80": dict(past=[70, 9], new=[5, 50], row=20, HD=80),
    "head_24": dict(past=[70, 9], new=[5, 5], row=2, HD=24), "f16": dict(past=[70, 9], new=[5, 1], row=5, dq=ir.F16),
}


class LostBlocks:
    """Block tables in whose lines, or whose free list, a block is none or lies past 32 bits of slots: its
    positions have no slot."""

    def __init__(self, table, free, past, new, block, M=4):
        self.past, self.new, self.block, self.M, self.free = past, new, block, M, free
        held = [-(-p // block) for p in past]
        self.tables = np.full((len(past), M), NONE, np.int64)
        for b, h in enumerate(held):
            self.tables[b, :h] = table[b][:h]
        self.held, self.T = held + [0], sum(new)

    def program(self):
        return tables_program(len(self.past), len(self.free), self.M, self.T, self.block)

    def values(self):
        return {"past": self.past, "new": self.new, "held": self.held, "free": self.free, "tables": self.tables}

    def slots(self):
        out, taken = [], 0
        for b, (p, n) in enumerate(zip(self.past, self.new)):
            line = list(self.tables[b][:self.held[b]])
            while len(line) * self.block < p + n:
                line.append(self.free[taken])
                taken += 1
            for pos in range(p, p + n):
                at = int(line[pos // self.block]) * self.block + pos % self.block
                out.append(NONE if line[pos // self.block] == NONE or at >= NONE else at)
        return out


LOST_BLOCKS = {
    "none_held": dict(table=[[NONE], [7]], free=[3, 4], past=[5, 6], new=[2, 3], block=16),
    "none_in_the_list": dict(table=[[9], [7]], free=[NONE, 4], past=[15, 16], new=[3, 2], block=16),
    "past_32_bits": dict(table=[[1 << 28], [(1 << 28) - 1]], free=[(1 << 28) + 1, (1 << 32) - 2], past=[5, 8], new=[2, 3], block=16),
    "past_32_bits_in_the_list": dict(table=[[1], [2]], free=[(1 << 28) + 1, (1 << 30) + 5], past=[15, 16], new=[9, 3], block=16),
    "the_last_slots": dict(table=[[(1 << 28) - 1], [0xFFFFFFFF // 24]], free=[5], past=[13, 10], new=[3, 9], block=16),
    "blocks_of_one": dict(table=[[NONE, NONE - 1], [5, 6]], free=[NONE - 1, NONE, 2], past=[2, 2], new=[1, 2], block=1),
    "odd_block": dict(table=[[0xFFFFFFFF // 24], [0xFFFFFFFF // 24 + 1]], free=[5], past=[10, 3], new=[9, 9], block=24),
}


def falling_starts(HD, dq=ir.BF16):
    """A batch of 64 rows, and starts that fall: 60 requests that claim all rows each, and single tokens
    over long caches among them. (Σ rows is 60 times what the batch holds.)"""
    past, new = [100] * 120 + [900] * 64, [0] * 120 + [1] * 64
    t = Batch(past=past, new=new, NKV=8, rep=4, HD=HD, BS=64, dq=dq)
    starts = [0, 64] * 60 + list(range(65))
    assert len(starts) == t.B + 1
    return t, starts


class Precision:
    """How many bits of a softmax weight reach the output. Keys and queries are small whole numbers over
    a power of two, so that every score is exact in 32 bits, at most 4.5, and what is left are the roundings
    of score · log2 e (2^-24 of up to 6.5), of 2^x (the hardware's last place), and of the sums over at
    most 90 keys: together below 2^-20 of an output's RMS for 24-bit weights. Weights of two bf16 terms
    are rounded at 2^-17 (RMS 2^-19 to 2^-18 of an output), of one at 2^-9 (2^-10)."""

    def __init__(self, new, dq, do, HD=64):
        g = np.random.default_rng(new)
        self.batch = t = Batch(past=[90 - new] * 3, new=[new] * 3, NKV=2, rep=4, HD=HD, BS=16, dq=dq, do=do, scale=2.0 ** -4)
        t.q = g.integers(-1, 2, t.q.shape).astype(float)
        t.kc = np.where(np.isnan(t.kc), np.nan, g.integers(-3, 4, t.kc.shape))
        t.q[:, :, 24:] = 0.0          # |scores| <= 24 · 3 / 16 = 4.5

    def rms(self, got):
        o, _ = self.batch.want()
        return float(np.sqrt(np.mean((got - o) ** 2) / np.mean(o ** 2)))

    def steps(self, got):
        """The error in units of half a step of the output's type at the exact value, the largest."""
        o, mag = self.batch.want()
        half = np.exp2(np.floor(np.log2(np.maximum(np.abs(o), 2.0 ** -14))) - (8 if self.batch.types[2] == ir.BF16 else 11))
        return float((np.abs(got - o) / (half + 2.0 ** -15 * mag)).max())

    def check(self, got, kind):
        if self.batch.types[2] == ir.F32:
            assert self.rms(got) < 2.0 ** -20, self.rms(got)
        elif self.batch.new[0] * self.batch.rep <= 32:
            # a few rows: 16 bits and more (2^-15 of the mean value, two times the weights' 2^-17 and as much
            # again for the rest), then one rounding
            assert self.steps(got) <= 1.0, self.steps(got)
        else:
            # many rows: one rounding of each weight to the cache's type, and the output's own; independent,
            # at most half a step each, RMS half a step / √3 at worst
            half = 2.0 ** -8 if self.batch.types[2] == ir.BF16 else 2.0 ** -11
            assert self.rms(got) < half * np.sqrt(2.0 / 3.0), self.rms(got)


PRECISION = {f"{'token' if n == 1 else 'drafts' if n < 9 else 'chunk'}_{x}_{y}": dict(new=n, dq=dq, do=do)
             for n in (1, 8, 40) for x, dq, y, do in (("bf16", ir.BF16, "f32", ir.F32), ("f16", ir.F16, "f32", ir.F32), ("bf16", ir.BF16, "bf16", ir.BF16), ("f16", ir.F16, "f16", ir.F16))}
HEADS = (16, 144, 176, 192, 208, 224, 240)


class SmallRoom(Batch):
    """A batch in a program whose intermediates leave the attention the smaller area for its partials:
    fewer runs of keys, and many rows that are not split or into few parts."""

    def program(self, **kw):
        p = super().program(**kw)
        x = p.pointwise("ballast", ir.map_(ir.ADD, p.input("ballast.in", (26 << 18,), ir.F32), ir.const(1.0)), ir.F32, role=3)
        p.pointwise("ballast.out", ir.map_(ir.ADD, x, ir.const(1.0)), ir.F32)
        return p


SMALL_ROOM = {
    "decodes": dict(past=[300 * i % 1700 for i in range(70)], new=[1] * 70, NKV=8, rep=4, HD=128, BS=16),
    "drafts": dict(past=[400 * i % 2100 for i in range(20)], new=[5] * 20, NKV=8, rep=4, HD=64, BS=32, dq=ir.F16),
    "mixed": dict(past=[900, 40, 9, 0, 77, 1500], new=[1, 90, 0, 33, 1, 8], NKV=8, rep=4, HD=128, BS=16, pad=9),
    "chunk": dict(past=[1500], new=[30], NKV=8, rep=4, HD=64, BS=16),
}


def huge_values(new, HD=64, requests=60):
    """bf16 values of 10^36 under scores that rise by 5 behind the first keys: the weights' sums, relative to
    the largest score, times the values stay within 32 bits' range (136 · 10^36), and so do the rows. So
    many requests that a workgroup goes over several tiles of keys."""
    t = Batch(past=[200] * requests, new=[new] * requests, NKV=8, rep=4, HD=HD, BS=16, scale=1.0)
    t.q[:] = 0.0
    t.q[:, :, 0] = 1.0
    j = np.arange(200 + new)
    for line in t.tables:
        at = (line[j // 16].astype(int), slice(None), j % 16)
        t.kc[at + (0,)] = np.where(j >= 64, 5.0, 0.0)[:, None]
        t.vc[at] = stored(1e36 * (1.0 + 0.1 * t.vc[at].clip(-3, 3)), ir.BF16)
    return t


def huge_far_values(new, HD=64, requests=1, dq=ir.BF16, value=2.0 ** 120):
    """Values of 2^120 at the first keys, whose scores are so far below the others that their weights are
    0 in 32 and in 64 bits: nothing of them is in any row."""
    t = Batch(past=[200] * requests, new=[new] * requests, NKV=8, rep=4, HD=HD, BS=16, dq=dq)
    t.q[:, :, 0] = 8.0
    j = np.arange(70)
    for line in t.tables:
        at = (line[j // 16].astype(int), slice(None), j % 16)
        t.kc[at + (0,)] = stored(-900.0 * HD ** 0.5, dq)
        t.vc[at] = value
    return t


HUGE_FAR = {"token": dict(new=1), "token_128": dict(new=1, HD=128), "drafts": dict(new=5), "chunk": dict(new=40), "tokens_60": dict(new=1, requests=60),
            "chunks_60": dict(new=12, requests=60), "head_24": dict(new=2, HD=24), "f32": dict(new=2, dq=ir.F32)}
