"""The operators where values, indices or lengths are at the edge of what they may be, on the GPU: the
cases of tests/test_cpu_operator_kernels.py again, and buffers of more than 2^32 elements."""
import numpy as np
import pytest

import paged_ref as ref
from paged_cases import HEADS, HUGE_FAR, LOST_BLOCKS, ODD_KEYS, ODD_QUERIES, ODD_VALUES, PRECISION, SMALL_ROOM, LostBlocks, OddKey, OddQuery, OddValue, Precision, SmallRoom, falling_starts, huge_far_values, huge_values
from sanic_amd import ir
from sanic_amd.backend import encode
from sanic_amd.program import NONE, Program
from test_gpu_operators import Batch, bind, read, stored, words

pytestmark = pytest.mark.gpu


def attention(dev, t):
    p = t.program()
    bufs = bind(dev, p, t.values())
    exe = dev.prepare(p)
    exe.execute_static(bufs)
    return read(p, bufs, "o"), exe.stage_kernel(0)


@pytest.mark.parametrize("case", ODD_VALUES)
def test_a_value_not_finite_in_the_past(dev, case):
    odd = OddValue(**ODD_VALUES[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", ODD_KEYS)
def test_a_key_of_minus_infinity_has_no_weight(dev, case):
    odd = OddKey(**ODD_KEYS[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", ODD_QUERIES)
def test_a_nan_in_a_query_is_in_its_row(dev, case):
    odd = OddQuery(**ODD_QUERIES[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", LOST_BLOCKS)
def test_lost_blocks_have_no_slots(dev, case):
    t = LostBlocks(**LOST_BLOCKS[case])
    p = t.program()
    bufs = bind(dev, p, t.values())
    dev.prepare(p).execute_static(bufs)
    assert words(p, bufs, "plan.slots").tolist() == t.slots()


@pytest.mark.parametrize("HD,dq", [(64, ir.BF16), (128, ir.F16), (24, ir.F32)])
def test_starts_that_fall_leave_nothing_behind(dev, HD, dq):
    """Nothing is written, and the next call (its arrivals are counted in the same words) is right."""
    t, starts = falling_starts(HD, dq)
    p = t.program()
    bufs = bind(dev, p, t.values())
    exe = dev.prepare(p)
    for _ in range(2):
        bufs["starts"].upload_array(np.asarray(starts, np.uint32))
        bufs["o"].upload(b"\xa5" * p.by_name["o"].nbytes)
        exe.execute_static(bufs)
        assert bufs["o"].download() == b"\xa5" * p.by_name["o"].nbytes
        bufs["starts"].upload_array(np.asarray(t.starts, np.uint32))
        exe.execute_static(bufs)
        t.check(read(p, bufs, "o"), exe.stage_kernel(0))


@pytest.mark.parametrize("case", PRECISION)
def test_bits_of_the_weights(dev, case):
    t = Precision(**PRECISION[case])
    t.check(*attention(dev, t.batch))


@pytest.mark.parametrize("HD", HEADS)
def test_every_head_size(dev, HD):
    for do in (ir.BF16, ir.F32):
        t = Batch(past=[190, 99], new=[1, 30], NKV=1, rep=2, HD=HD, BS=16, do=do)
        t.check(*attention(dev, t))


@pytest.mark.parametrize("case", SMALL_ROOM)
def test_little_room_for_partials(dev, case):
    t = SmallRoom(**SMALL_ROOM[case])
    p = t.program()
    bufs = bind(dev, p, {**t.values(), "ballast.in": np.zeros(p.by_name["ballast.in"].shape)})
    exe = dev.prepare(p)
    for _ in range(2):
        exe.execute_static(bufs)
        t.check(read(p, bufs, "o"), exe.stage_kernel(0))


@pytest.mark.parametrize("new,HD", [(1, 64), (5, 128), (12, 64)])
def test_values_near_the_end_of_the_range(dev, new, HD):
    t = huge_values(new, HD)
    t.check(*attention(dev, t))


@pytest.mark.parametrize("case", HUGE_FAR)
def test_huge_values_without_weight(dev, case):
    t = huge_far_values(**HUGE_FAR[case])
    t.check(*attention(dev, t))


@pytest.mark.parametrize("dtype", [ir.BF16, ir.F32])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_caches_past_32_bits_of_elements(dev, dtype, order):
    """Blocks at both ends of pools of 4.6·10^9 elements: written through slots, then read."""
    NB, NKV, BS, HD, NH, T = 70000, 8, 64, 128, 16, 75
    past, new = [0, 0, 0], [70, 1, 4]
    tables = np.array([[NB - 1, 3], [65536, NONE], [NB - 2, NONE]])
    p = Program()
    shape = (NB, NKV, BS, HD) if order == "heads" else (NB, BS, NKV, HD)
    caches = [p.state(n, shape, dtype) for n in ("kc", "vc")]
    if order == "tokens":
        caches = [ir.permute(c, (0, 2, 1, 3)) for c in caches]
    starts = p.input("starts", (4,), ir.U32)
    p.cache_write("write", p.input("k", (T, NKV, HD), dtype), p.input("v", (T, NKV, HD), dtype), p.input("slots", (T,), ir.U32), starts, *caches)
    p.paged_attention("o", p.input("q", (T, NH, HD), dtype), *caches, p.input("tables", (3, 2), ir.U32), starts, p.input("past", (3,), ir.U32), out_dtype=dtype)
    g = np.random.default_rng(4)
    q, k, v = (stored(g.standard_normal((T, h, HD)), dtype) for h in (NH, NKV, NKV))
    slots = [int(tables[b][i // BS]) * BS + i % BS for b in range(3) for i in range(new[b])]
    assert max(slots) * NKV * HD > 1 << 32
    vals = {"q": q, "k": k, "v": v, "slots": slots, "starts": np.concatenate(([0], np.cumsum(new))), "tables": tables, "past": past}
    bufs = {b.name: dev.from_values(vals[b.name], b.dtype) if b.name in vals else dev.alloc(b.nbytes) for b in p.buffers}
    exe = dev.prepare(p)
    exe.execute_static(bufs)
    # the same batch over a pool of its blocks alone
    t = Batch(past=past, new=new, NKV=NKV, rep=NH // NKV, HD=HD, BS=BS, dq=dtype)
    t.tables = np.array([[0, 1], [2, NONE], [3, NONE]])
    t.kc, t.vc, t.q = np.zeros((4, NKV, BS, HD)), np.zeros((4, NKV, BS, HD)), q
    row = 0
    for b in range(3):
        for i in range(new[b]):
            t.kc[t.tables[b][i // BS], :, i % BS], t.vc[t.tables[b][i // BS], :, i % BS] = k[row], v[row]
            row += 1
    t.check(read(p, bufs, "o"), exe.stage_kernel(1))


def test_probabilities_past_32_bits_of_elements(dev):
    """Requests in the last rows of [40000, 128256]: rows from 5.1·10^9 elements on."""
    T, V, B, n = 40000, 128256, 2, 10
    g = np.random.default_rng(9)
    p = Program()
    p.verify_drafts("check", p.input("p", (T, V), ir.BF16), None, *(p.input(name, shape, dt) for name, shape, dt in (
        ("tokens", (T,), ir.U32), ("starts", (B + 1,), ir.U32), ("u", (T,), ir.F32), ("draw", (B,), ir.F32))))
    probs = g.random((n, V)) ** 8
    probs = stored(probs / probs.sum(1, keepdims=True), ir.BF16)
    tokens, u, draw = np.zeros(T, np.int64), np.zeros(T), stored(g.random(B), ir.F32)
    tokens[T - n:] = g.integers(0, V, n)
    tokens[T - n + 1], tokens[T - n + 2] = probs[0].argmax(), probs[1].argmax()
    u[T - n:] = stored(probs[np.arange(n - 1), tokens[T - n + 1:]].max() * 0.5, ir.F32)
    starts = [T - n, T - n + 6, T]
    vals = {"tokens": tokens, "starts": starts, "u": u, "draw": draw}
    bufs = {b.name: dev.from_values(vals[b.name], b.dtype) if b.name in vals else dev.alloc(b.nbytes) for b in p.buffers}
    bufs["p"].slice((T - n) * V * 2, n * V * 2).upload(encode(probs, ir.BF16))
    dev.prepare(p).execute_static(bufs)
    want, accepted = ref.verify(probs, None, tokens[T - n:], [0, 6, n], u[T - n:], draw)
    assert words(p, bufs, "check.accepted").tolist() == accepted and accepted[0] > 0
    assert words(p, bufs, "check.tokens")[T - n:].tolist() == want
