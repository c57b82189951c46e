"""The operators' generated kernels themselves, on the CPU (wave_host.py): every address, LDS index, wait
and work item of the text that the GPU runs, over ragged and mixed batches, with the workgroups in
different orders; results against tests/paged_ref.py, arrival counters back at zero."""
import os
import random
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import paged_ref as ref
import wave_host as host
from paged_cases import HEADS, HUGE_FAR, LOST_BLOCKS, ODD_KEYS, ODD_QUERIES, ODD_VALUES, PRECISION, SMALL_ROOM, LostBlocks, OddKey, OddQuery, OddValue, Precision, SmallRoom, falling_starts, huge_far_values, huge_values
from sanic_amd import ir
from sanic_amd.backend import decode, encode
from sanic_amd.program import NONE
from test_gpu_operators import ATTN, Batch, stored, tables_program, verify_program, write_program

pytestmark = pytest.mark.skipif(not host.available(), reason="no host compiler for the kernels' dialect")

ORDERS = (0, 5)        # workgroups forwards, shuffled


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tmp_path_factory.mktemp("kernels")


@pytest.fixture(scope="module")
def results(request, folder):
    """The module's selected cases that run by themselves, on every CPU: test name -> future."""
    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        out = {}
        for item in request.session.items:
            alone = getattr(getattr(item, "function", None), "alone", None)
            if alone and item.name not in out and item.module is request.module:
                run_in = folder / item.name.replace("/", "_")
                run_in.mkdir()
                out[item.name] = pool.submit(alone, *item.callspec.params.values(), folder, run_in)
        yield out
        pool.shutdown(cancel_futures=True)


def run_alone(body):
    """A test whose cases `results` runs side by side."""
    def mark(test):
        test.alone = body
        return test
    return mark


def attention(t, folder, run_in, starts=None, order=0, math=True, change=lambda text: text, **kw):
    """The batch's output [T, NH, HD] and the kernel's kind; fails where the kernel goes out of bounds."""
    kind, source = t.program(**kw).emit(0)
    c = host.constants(source)
    dq, dc, do = t.types
    q, kc, vc = t.q, t.kc, t.vc
    if kw.get("order") == "tokens":
        kc, vc = kc.transpose(0, 2, 1, 3), vc.transpose(0, 2, 1, 3)
    if kw.get("q_order") == "heads":
        q = q.transpose(1, 0, 2)
    ops, grid = host.attention_operands(c, encode(q, dq), encode(kc, dc), encode(vc, dc), t.tables, t.starts if starts is None else starts,
                                        t.past, t.q.size * ir.dtype_bytes(do, 1))
    why = host.run(host.build(source, str(folder), math, change), str(run_in), grid, ops, order)
    assert why is None, why
    if len(ops) > 7:
        assert not any(ops[8]), "arrivals are left over for the next launch"
    n = min(int(t.starts[-1]), t.T) * t.NKV * t.rep * t.HD * ir.dtype_bytes(do, 1)
    assert ops[6][n:] == b"\xa5" * (len(ops[6]) - n), "rows behind the last request were written"
    return decode(bytes(ops[6]), do, t.q.size).reshape(t.q.shape), kind


def _every_order(case, folder, run_in):
    t = Batch(**ATTN[case])
    first = None
    for order in ORDERS:
        got, kind = attention(t, folder, run_in, order=order)
        t.check(got, kind)
        assert first is None or got.tobytes() == first.tobytes(), "the order of the workgroups changes the result"
        first = got


@run_alone(_every_order)
@pytest.mark.parametrize("case", ATTN)
def test_attention_on_the_cpu(case, results, request):
    results[request.node.name].result()


@pytest.mark.parametrize("order,q_order", [("tokens", "tokens"), ("heads", "heads"), ("tokens", "heads")])
@pytest.mark.parametrize("HD", [64, 112])
def test_attention_orders_on_the_cpu(order, q_order, HD, folder, tmp_path):
    t = Batch(past=[70, 200, 4], new=[40, 1, 3], NKV=2, rep=4, HD=HD, BS=16)
    t.check(*attention(t, folder, tmp_path, order=order, q_order=q_order))


def _mixed(seed):
    """A batch of decodes, drafts, chunks and idle requests, some cut off at T."""
    r = random.Random(seed)
    B = r.choice([1, 2, 5, 17, 41, 63, 64, 65, 130])
    NKV, rep, HD = r.choice([1, 2, 4, 8]), r.choice([1, 2, 4, 7, 8]), r.choice([16, 64, 80, 128, 128, 144, 208])
    new = [r.choice([0, 1, 1, 1, r.randint(2, 9), r.randint(10, 90)]) for _ in range(B)]
    if r.random() < 0.6:
        new[r.randrange(B)] = r.randint(100, 700)
    new[0] = max(new[0], 1)
    past = [r.choice([0, r.randint(1, 70), r.randint(100, 1500)]) for _ in range(B)]
    t = Batch(past=past, new=new, NKV=NKV, rep=rep, HD=HD, BS=r.choice([1, 8, 16, 16, 24, 32, 64]), window=r.choice([0, 0, r.randint(1, 900)]),
              pad=r.choice([0, 7]), seed=seed, dq=r.choice([ir.BF16, ir.F16]))
    for _ in range(r.randint(0, 3)):      # blocks that are gone
        t.tables[r.randrange(B), r.randrange(t.M)] = r.choice([NONE, t.NB, t.NB + 1])
    starts = t.starts
    if r.random() < 0.3 and t.T > 4:      # rows that do not fit
        t.T -= 3
        t.q = t.q[:t.T]
    return t, starts


def _in_bounds(seed, folder, run_in):
    t, starts = _mixed(seed)
    attention(t, folder, run_in, starts, order=seed, math=False)


@run_alone(_in_bounds)
@pytest.mark.parametrize("seed", range(24))
def test_mixed_batches_stay_in_bounds(seed, results, request):
    results[request.node.name].result()


def test_what_the_host_run_notices(folder, tmp_path):
    """A buffer that ends early, a tile read before it has arrived, a part of LDS that is not there."""
    t = Batch(**ATTN["decode"])
    with pytest.raises(AssertionError, match="operand 1 at byte"):
        kc = t.kc
        t.kc = kc[:int(t.tables[0, 0])]     # the pool ends ahead of a block in use
        attention(t, folder, tmp_path)
    t.kc = kc
    for old, new, said in (("wh::turn_barrier(0)", "wh::turn_barrier(99)", None),
                           ("n * 512], 16, 0, 0)", "n * 512 + RING], 16, 0, 0)", "signal 4|outside its ring")):
        def change(text):
            assert old in text
            return text.replace(old, new)
        with pytest.raises(AssertionError, match=said):
            t.check(*attention(t, folder, tmp_path, change=change))


@pytest.mark.parametrize("HD,dq", [(64, ir.BF16), (128, ir.F16), (24, ir.F32)])
def test_starts_that_fall_leave_nothing_behind(HD, dq, folder, tmp_path):
    """Overlapping requests can be more work than the launch has workgroups: nothing is begun."""
    t, starts = falling_starts(HD, dq)
    t.starts = np.zeros(t.B + 1, np.int64)      # every row is to be left as it was
    attention(t, folder, tmp_path, starts, math=False)


def _end_of_the_range(new, HD, folder, run_in):
    t = huge_values(new, HD)
    t.check(*attention(t, folder, run_in))


@run_alone(_end_of_the_range)
@pytest.mark.parametrize("new,HD", [(1, 64), (5, 128), (12, 64)])
def test_values_near_the_end_of_the_range(new, HD, results, request):
    results[request.node.name].result()


def _huge_far(case, folder, run_in):
    t = huge_far_values(**HUGE_FAR[case])
    t.check(*attention(t, folder, run_in))


@run_alone(_huge_far)
@pytest.mark.parametrize("case", HUGE_FAR)
def test_huge_values_without_weight(case, results, request):
    results[request.node.name].result()


def _odd_value(case, folder, run_in):
    odd = OddValue(**ODD_VALUES[case])
    odd.check(*attention(odd.batch, folder, run_in))


@run_alone(_odd_value)
@pytest.mark.parametrize("case", ODD_VALUES)
def test_a_value_not_finite_in_the_past(case, results, request):
    results[request.node.name].result()


def _odd_key(case, folder, run_in):
    odd = OddKey(**ODD_KEYS[case])
    odd.check(*attention(odd.batch, folder, run_in))


@run_alone(_odd_key)
@pytest.mark.parametrize("case", ODD_KEYS)
def test_a_key_of_minus_infinity_has_no_weight(case, results, request):
    results[request.node.name].result()


def _odd_query(case, folder, run_in):
    odd = OddQuery(**ODD_QUERIES[case])
    odd.check(*attention(odd.batch, folder, run_in))


@run_alone(_odd_query)
@pytest.mark.parametrize("case", ODD_QUERIES)
def test_a_nan_in_a_query_is_in_its_row(case, results, request):
    results[request.node.name].result()


def _precision(case, folder, run_in):
    """Passes, and would not with a term of the weights less."""
    t = Precision(**PRECISION[case])
    t.check(*attention(t.batch, folder, run_in))
    name = "FEW_TERMS" if t.batch.new[0] * t.batch.rep <= 32 else "MANY_TERMS"
    terms = host.constants(t.batch.program().emit(0)[1])[name]
    if terms > 1 and t.batch.types[0] == ir.BF16:
        less = lambda text: text.replace(f"constexpr int {name} = {terms};", f"constexpr int {name} = {terms - 1};")  # noqa: E731
        with pytest.raises(AssertionError):
            t.check(*attention(t.batch, folder, run_in, change=less))


@run_alone(_precision)
@pytest.mark.parametrize("case", PRECISION)
def test_bits_of_the_weights(case, results, request):
    results[request.node.name].result()


def _heads(HD, folder, run_in):
    for do in (ir.BF16, ir.F32):
        t = Batch(past=[190, 99], new=[1, 30], NKV=1, rep=2, HD=HD, BS=16, do=do)
        t.check(*attention(t, folder, run_in))


@run_alone(_heads)
@pytest.mark.parametrize("HD", HEADS)
def test_every_head_size_on_the_cpu(HD, results, request):
    results[request.node.name].result()


def _small_room(case, folder, run_in):
    t = SmallRoom(**SMALL_ROOM[case])
    roomy, tight = (host.constants(p.emit(0)[1]) for p in (Batch.program(t), t.program()))
    assert tight["SLOTS"] * 4 < roomy["SLOTS"]
    t.check(*attention(t, folder, run_in))


@run_alone(_small_room)
@pytest.mark.parametrize("case", SMALL_ROOM)
def test_little_room_for_partials(case, results, request):
    results[request.node.name].result()


def _words(x):
    return bytearray((np.asarray(x, np.int64) & 0xFFFFFFFF).astype(np.uint32).tobytes())


def _numbers(x):
    return np.frombuffer(bytes(x), np.uint32).astype(np.int64)


@pytest.mark.parametrize("B,seed", [(1, 0), (5, 1), (64, 2), (257, 3)])
def test_block_tables_on_the_cpu(B, seed, folder, tmp_path):
    r = np.random.default_rng(seed)
    block, M, past = 8, 12, r.integers(0, 70, B)
    new = np.where(r.random(B) < 0.3, 0, r.integers(1, 40, B))
    held = list(-(-past // block) + (r.random(B) < 0.2)) + [2]
    F, T = int(r.integers(B, 4 * B + 9)), int(new.sum()) + 9
    free = r.permutation(F + B * M)
    tables = np.full((B, M), NONE, np.int64)
    for b in range(B):
        tables[b, :held[b]] = free[F + b * M:F + b * M + held[b]]
    source = tables_program(B, F, M, T, block).emit(0)[1]
    ops = [bytes(_words(past)), bytes(_words(new)), bytes(_words(held)), bytes(_words(free[:F])), _words(tables), bytearray(4 * T), bytearray(4 * T),
           bytearray(4 * B + 4), bytearray(4 * B + 4)]
    why = host.run(host.build(source, str(folder)), str(tmp_path), min((max(T, B + 1) + 255) // 256, 512), ops, order=seed)
    assert why is None, why
    starts, slots, positions, after, want = ref.block_tables(past, new, held, free[:F], tables, block, T)
    n = starts[-1]
    assert _numbers(ops[8]).tolist() == starts and _numbers(ops[5])[:n].tolist() == slots and _numbers(ops[6])[:n].tolist() == positions
    assert _numbers(ops[7]).tolist() == [int(x) for x in after] and (_numbers(ops[4]).reshape(B, M) == want).all()


@pytest.mark.parametrize("case", LOST_BLOCKS)
def test_lost_blocks_have_no_slots(case, folder, tmp_path):
    t = LostBlocks(**LOST_BLOCKS[case])
    v, B = t.values(), len(t.past)
    ops = [bytes(_words(v[n])) for n in ("past", "new", "held", "free")] + [_words(t.tables)] + [bytearray(4 * n) for n in (t.T, t.T, B + 1, B + 1)]
    why = host.run(host.build(t.program().emit(0)[1], str(folder)), str(tmp_path), 1, ops)
    assert why is None, why
    assert _numbers(ops[5]).tolist() == t.slots()


@pytest.mark.parametrize("HD,order,fused", [(16, "heads", False), (7, "tokens", False), (24, "tokens", True)])
def test_cache_write_on_the_cpu(HD, order, fused, folder, tmp_path):
    T, NKV, NB, BS, B = 21, 3, 5, 8, 2
    g = np.random.default_rng(HD)
    source = write_program(T, NKV, HD, NB, BS, B, ir.F32, ir.BF16, order, fused).emit(0)[1]
    slots = g.permutation(NB * BS)[:T]
    slots[[0, 3]] = NONE, NB * BS
    k, v = g.standard_normal((2, T, NKV, HD))
    kv = np.concatenate((k.reshape(T, -1), np.zeros((T, 8)), v.reshape(T, -1)), 1)
    src = [encode(kv, ir.F32)] * 2 if fused else [encode(k, ir.F32), encode(v, ir.F32)]
    caches = [bytearray(encode(np.full((NB, BS, NKV, HD), 3.0), ir.BF16)) for _ in "kv"]
    ops = [*src, bytes(_words(slots)), bytes(_words([0, 4, 19])), *caches]
    why = host.run(host.build(source, str(folder)), str(tmp_path), 4, ops)
    assert why is None, why
    for got, rows in zip(ops[4:], (k, v)):
        want = np.full((NB * BS, NKV, HD), 3.0)
        live = [r for r in range(19) if slots[r] < NB * BS]
        want[slots[live]] = stored(stored(rows[live], ir.F32), ir.BF16)
        got = decode(bytes(got), ir.BF16, want.size)
        want = want.reshape(NB, BS, NKV, HD)
        np.testing.assert_array_equal(got.reshape(want.shape) if order == "tokens" else got.reshape(NB, NKV, BS, HD).transpose(0, 2, 1, 3), want)


@pytest.mark.parametrize("V,dp,dq", [(1, ir.F32, ir.F32), (2049, ir.BF16, ir.F32), (9001, ir.F32, None), (50021, ir.BF16, None)])
def test_verify_on_the_cpu(V, dp, dq, folder, tmp_path):
    g = np.random.default_rng(V)
    counts = [5, 1, 0, 9, 3, 2]
    T, B = sum(counts) + 2, len(counts)
    e = np.exp(g.standard_normal((T, V)) * 2)
    p = e / e.sum(1, keepdims=True)
    e *= np.exp(0.5 * g.standard_normal((T, V)))
    q = e / e.sum(1, keepdims=True)
    p, u, draw = stored(p, dp), stored(g.random(T), ir.F32), stored(g.random(B), ir.F32)
    q = None if dq is None else stored(q, dq)
    tokens, starts = g.integers(0, V, T), np.concatenate(([0], np.cumsum(counts)))
    tokens[1:] = [int(g.choice(V, p=x / x.sum())) for x in (p if q is None else q)[:-1]]
    source = verify_program(T, B, V, dp, dq).emit(0)[1]
    c = host.constants(source)
    ops = [encode(p, dp), encode(p if q is None else q, dp if q is None else dq), bytes(_words(tokens)), encode(u, ir.F32), encode(draw, ir.F32),
           bytes(_words(starts)), bytearray(4 * B), _words([7] * T), bytearray(b"\xff" * (B * ((c["CHUNKS"] + 15) // 16 * 16) * 8)), bytearray(8 * c["CSTRIDE"] * 4)]
    for order in ORDERS:
        why = host.run(host.build(source, str(folder)), str(tmp_path), (B + 7) // 8 * 8 * c["CHUNKS"], ops, order)
        assert why is None, why
        want, accepted = ref.verify(p, q, tokens, starts, u, draw)
        assert _numbers(ops[6]).tolist() == accepted and _numbers(ops[7]).tolist() == want + [7, 7] and not any(ops[9])
