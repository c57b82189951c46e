"""The operators together as a serving loop runs them: block tables, cache write and attention of one
step in one program (configs.paged_step), drafts verified behind it (configs.draft_verification),
several steps over one cache; and how such programs run: execute_static, capture, refusals."""
import numpy as np
import pytest

import paged_ref as ref
from sanic_amd import carrier as C
from sanic_amd import configs, ir
from sanic_amd.abi import SanicError
from sanic_amd.graph import Graph
from sanic_amd.program import NONE, STREAM, Program
from test_gpu_operators import FILL, HALF, Batch, bind, read, stored, tables_program, words

pytestmark = pytest.mark.gpu


def rope(x, pos, theta=500000.0):
    """Rotate-half RoPE of rows [T, heads, HD] at their positions, f64."""
    half = x.shape[-1] // 2
    a = np.asarray(pos, np.float64)[:, None, None] * theta ** (-np.arange(half) / half)
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate((lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)), -1)


@pytest.mark.parametrize("how", ["execute_static", "capture"])
@pytest.mark.parametrize("HD,window", [(64, 0), (128, 40)])
def test_serving_steps(dev, how, HD, window):
    """Prompts in chunks, decodes, drafts of which some are taken back, an idle request and one that
    runs out of blocks: each step's tables, caches and attention against the definitions."""
    T, B, NH, NKV, NB, BS, M = 96, 5, 8, 2, 40, 16, 12
    p = configs.paged_step(T, B, NH, NKV, HD, NB, BS, M, window=window)
    g = np.random.default_rng(HD)
    free = g.permutation(NB)
    # the caches hold NaN where nothing has been written
    vals = {"tables": np.full((B, M), NONE), "k_cache": np.full((NB, NKV, BS, HD), np.nan), "v_cache": np.full((NB, NKV, BS, HD), np.nan),
            "free": free, "held": np.zeros(B + 1), "past": np.zeros(B), "new": np.zeros(B)}
    for n, w in (("q", NH), ("k", NKV), ("v", NKV)):
        vals[n] = np.zeros((T, w * HD))
    bufs = bind(dev, p, vals)
    exe = dev.prepare(p)
    out = dict(bufs)
    if how == "capture":
        state = {b.name for b in p.buffers if b.role in (0, 1)}
        replay = exe.capture({n: b for n, b in bufs.items() if n in state}, [("plan.held", "held")])
        out.update({b.name: replay.buffer(b.name) for b in p.buffers if b.role == 2})
        for b in p.buffers:
            if b.role == 2:
                out[b.name].upload(b"\xa5" * b.nbytes)
    past, held, tables = np.zeros(B, np.int64), [0] * (B + 1), np.full((B, M), NONE, np.int64)
    kc, vc = np.full((NB, NKV, BS, HD), np.nan), np.full((NB, NKV, BS, HD), np.nan)
    steps = [([40, 20, 0, 3, 33], 0), ([30, 1, 0, 5, 33], 2), ([1, 1, 60, 5, 20], 3), ([1, 0, 0, 5, 90], 1), ([1, 1, 1, 5, 1], 0), ([1, 1, 1, 5, 0], 0)]
    for new, back in steps:
        rows = {n: stored(g.standard_normal((T, w, HD)), ir.BF16) for n, w in (("q", NH), ("k", NKV), ("v", NKV))}
        for n in ("past", "new"):
            bufs[n].upload_array(np.asarray(past if n == "past" else new, np.uint32))
        for n in rows:
            bufs[n].upload(_bf16(rows[n]))
        if how == "execute_static":
            bufs["held"].upload_array(np.asarray(held, np.uint32))
            exe.execute_static(bufs)
        else:
            replay.step()
        starts, slots, positions, held, tables = ref.block_tables(past, new, held, free, tables, BS, T)
        n = starts[-1]
        assert words(p, out, "plan.starts").tolist() == starts and words(p, out, "plan.slots")[:n].tolist() == slots
        assert words(p, out, "plan.positions")[:n].tolist() == positions and words(p, out, "plan.held").tolist() == held
        np.testing.assert_array_equal(words(p, bufs, "tables"), tables)
        if how == "capture":
            assert words(p, bufs, "held").tolist() == held       # fed back inside the graph
        # a rotated row in f32 lies within a few of its steps of the f64 value (angles up to 100 rad by
        # frequencies that are exp() of f32: 2^-19 of the angle and the hardware sine's 2^-20), then one
        # bf16 rounding
        kr, qr = rope(rows["k"][:n], positions), rope(rows["q"][:n], positions)
        got_k, got_v = read(p, bufs, "k_cache"), read(p, bufs, "v_cache")
        for r in range(n):
            if slots[r] != NONE:
                at = (slots[r] // BS, slice(None), slots[r] % BS)
                kc[at], vc[at] = kr[r], rows["v"][r]
        np.testing.assert_array_equal(np.isnan(got_k), np.isnan(kc))
        ok = ~np.isnan(kc)
        assert (np.abs(got_k - kc)[ok] <= HALF[ir.BF16] * np.abs(kc)[ok] + 2.0 ** -9 * 2.0 ** -3).all()
        np.testing.assert_array_equal(got_v, vc)
        # attention from the device's own cache, so that only q's rotation is added to its own
        # tolerance: two roundings of q (its f32 rotation is far below) scale the scores by 2^-8
        t = Batch(past=[0] * B, new=[1] * B, NKV=NKV, rep=NH // NKV, HD=HD, BS=BS, window=window)
        q16 = stored(qr, ir.BF16)
        t.q, t.kc, t.vc, t.tables, t.past, t.starts, t.T = q16, got_k, got_v, tables, past, np.array(starts), n
        o, mag = t.want()
        got = read(p, out, "o").reshape(T, NH, HD)[:n]
        # a q element that rounds the other way moves a score by at most 2^-8·Σ|q·k|·scale over the few
        # such elements; half of the row's sum is far more than occur
        s = 2.0 ** -8 * 0.5 * HD / np.sqrt(HD)
        assert (np.abs(got - o) <= HALF[ir.BF16] * np.abs(o) + (2 * HALF[ir.BF16] + 2 * s) * mag + 1e-6).all()
        past = past + np.diff(starts)
        past = np.maximum(past - np.where(np.asarray(new) == 5, back, 0), 0)     # rejected drafts


def _bf16(v):
    from sanic_amd.backend import encode
    return encode(v, ir.BF16)


def test_attention_follows_the_captured_cache(dev):
    """Replays of one graph see what the host changed in the bound buffers between them, and two
    graphs of one program keep to their own workspaces."""
    t = Batch(past=[900, 40], new=[1, 5], NKV=2, rep=4, HD=64, BS=16)
    p = t.program()
    exe = dev.prepare(p)
    sets = []
    for seed in (1, 2):
        u = Batch(past=[900, 40], new=[1, 5], NKV=2, rep=4, HD=64, BS=16, seed=seed)
        bufs = bind(dev, p, u.values())
        sets.append((u, bufs, exe.capture({n: b for n, b in bufs.items() if n != "o"})))
    want = []
    for u, bufs, _ in sets:
        exe.execute_static(bufs)
        want.append(bufs["o"].download())
    for turn in range(4):
        for (u, bufs, replay), w in zip(sets, want):
            replay.step_many(3)
            got = replay.buffer("o").download()
            n = int(u.starts[-1]) * 8 * 64 * 2
            assert got[:n] == w[:n]
            exe.execute_static(bufs)
            assert bufs["o"].download()[:n] == w[:n]
    # another past in the same buffers
    u, bufs, replay = sets[0]
    u.past = [700, 3]
    bufs["past"].upload_array(np.asarray(u.past, np.uint32))
    replay.step()
    out = replay.buffer("o").read(ir.BF16, u.q.size).reshape(u.q.shape)
    u.check(out, exe.stage_kernel(0))


def test_two_devices_handles_take_turns(dev):
    """execute_static from two handles on one GPU shares the static workspace, one call after the other."""
    from sanic_amd.backend import HipDevice
    other = HipDevice(0)
    try:
        work = []
        for d, seed in ((dev, 3), (other, 4)):
            t = Batch(past=[3000, 900], new=[1, 1], NKV=2, rep=4, HD=64, BS=16, seed=seed)
            p = t.program()
            work.append((t, p, bind(d, p, t.values()), d.prepare(p)))
        for _ in range(20):
            for t, p, bufs, exe in work:
                exe.execute_static(bufs)
        for t, p, bufs, exe in work:
            t.check(read(p, bufs, "o"), exe.stage_kernel(0))
    finally:
        del work, bufs, exe, p, t
        other.close()


def test_drafts_from_logits(dev):
    T, B, V = 17, 4, 5003
    p = configs.draft_verification(T, B, V, temperature=0.8)
    g = np.random.default_rng(11)
    logits = stored(g.standard_normal((T, V)) * 2, ir.F32)
    z = logits / 0.8
    probs = np.exp(z - z.max(1, keepdims=True))
    probs /= probs.sum(1, keepdims=True)
    drafts = logits + 0.4 * g.standard_normal((T, V))
    q = np.exp(drafts - drafts.max(1, keepdims=True))
    q = stored(q / q.sum(1, keepdims=True), ir.F32)
    tokens = np.array([g.choice(V, p=r / r.sum()) for r in q])
    tokens[1:] = tokens[:-1].copy()
    vals = {"logits": logits, "draft_probs": q, "tokens": tokens, "starts": [0, 5, 6, 12, 17], "u": stored(g.random(T), ir.F32),
            "draw": stored(g.random(B), ir.F32)}
    bufs = bind(dev, p, vals)
    dev.prepare(p).execute_static(bufs)
    want, accepted = ref.verify(probs, q, tokens, vals["starts"], vals["u"], vals["draw"])
    # f32 probabilities are 2^-20 off the f64 ones at most (exponent of |z| < 16, a sum of 5003): the
    # inputs of this seed keep every test and every drawn sum further than 2^-16 from its border
    for b in range(B):
        for r in range(vals["starts"][b], vals["starts"][b + 1] - 1):
            x = tokens[r + 1]
            assert abs(vals["u"][r] * q[r, x] / probs[r, x] - 1) > 2.0 ** -16
    assert words(p, bufs, "check.accepted").tolist() == accepted
    assert words(p, bufs, "check.tokens").tolist() == want


# ── refusals of a call ───────────────────────────────────────────────────────

def _tables_call(dev):
    p = tables_program(2, 9, 4, 6, 16)
    vals = {"past": [3, 0], "new": [1, 5], "held": [1, 0, 0], "free": np.arange(9), "tables": np.full((2, 4), NONE)}
    return p, dev.prepare(p), bind(dev, p, vals)


def test_execute_refuses_programs_that_write_states(dev):
    p, exe, bufs = _tables_call(dev)
    with pytest.raises(SanicError) as e:
        exe.execute({n: b for n, b in bufs.items() if not n.startswith("plan.")})
    assert e.value.code == 8


def test_execute_static_still_refuses_pointwise_states(dev):
    p, _, bufs = _tables_call(dev)
    c = p.state("count", (), ir.F32)
    p.pointwise("count.next", ir.map_(ir.ADD, c, ir.const(1.0)), ir.F32, grid=(), into="count")
    exe = dev.prepare(p)
    with pytest.raises(SanicError) as e:
        exe.execute_static({**bufs, "count": dev.from_values([0.0], ir.F32)})
    assert e.value.code == 8


@pytest.mark.parametrize("a,b", [("plan.held", "held"), ("plan.slots", "plan.positions"), ("tables", "free"), ("plan.starts", "past")])
def test_overlapping_buffers_are_refused(dev, a, b):
    p, exe, bufs = _tables_call(dev)
    at = dev.alloc(4096)
    bufs = dict(bufs)
    na, nb = p.by_name[a].nbytes, p.by_name[b].nbytes
    bufs[a], bufs[b] = at.slice(256, na), at.slice(256 + na - 4, nb)      # one word in common
    with pytest.raises(SanicError) as e:
        exe.execute_static(bufs)
    assert e.value.code == 7 and "overlap" in str(e.value)
    with pytest.raises(SanicError):
        exe.capture({n: x for n, x in bufs.items() if not n.startswith("plan.")}) if "plan." not in a + b else exe.execute_static(bufs)
    bufs[b] = at.slice(256 + na, nb)                                       # behind each other
    bufs[b].upload_array(np.zeros(nb // 4, np.uint32))
    bufs[a].upload_array(np.zeros(na // 4, np.uint32))
    exe.execute_static(bufs)
    dev.sync()


def test_odd_addresses_are_refused(dev):
    p, exe, bufs = _tables_call(dev)
    at = dev.alloc(4096)
    with pytest.raises(SanicError) as e:
        exe.execute_static({**bufs, "past": dev.wrap(at.device_ptr + 2, 8)})
    assert e.value.code == 7


@pytest.mark.parametrize("offset", [4, 8, 12])
def test_buffers_at_any_word(dev, offset):
    """Operands at addresses that are no multiple of 16."""
    for t in (Batch(past=[300, 40], new=[1, 5], NKV=2, rep=4, HD=64, BS=16), Batch(past=[30, 40], new=[70, 5], NKV=1, rep=4, HD=128, BS=16)):
        p = t.program()
        bufs = bind(dev, p, t.values())
        moved, keep = {}, []
        for n, b in bufs.items():
            big = dev.alloc(b.nbytes + 64)
            keep.append(big)
            moved[n] = big.slice(offset, b.nbytes)
            moved[n].upload(b.download())
        exe = dev.prepare(p)
        exe.execute_static(moved)
        t.check(read(p, moved, "o"), exe.stage_kernel(0))


def test_feedback_of_whole_numbers_keeps_all_bits(dev):
    """A u32 that is fed back into a u32 does not pass through a float."""
    p, exe, bufs = _tables_call(dev)
    big = [(1 << 24) + 1, 0, 0x80000001]
    bufs["held"].upload_array(np.asarray([1, 0, 0], np.uint32))
    bufs["past"].upload_array(np.asarray([3, 0], np.uint32))
    replay = exe.capture({n: b for n, b in bufs.items() if not n.startswith("plan.")}, [("plan.held", "held")])
    # nobody brings rows, so `held` goes through as it is
    bufs["new"].upload_array(np.zeros(2, np.uint32))
    bufs["held"].upload_array(np.asarray(big, np.uint32))
    for _ in range(3):
        replay.step()
        assert words(p, bufs, "held").tolist() == big


def test_graph_machine_over_operators(dev):
    """Graph.update feeds `held` back; the machine's states start at zero, so every table entry must
    be written before it is read."""
    g = Graph()
    p = g.program
    B, T, M, BS, F = 3, 30, 6, 4, 16
    g.state("tables", (B, M), ir.U32)
    held = g.state("held", (B + 1,), ir.U32)
    plan = p.block_tables("plan", g.input("past", (B,), ir.U32), g.input("new", (B,), ir.U32), held, g.input("free", (F,), ir.U32), "tables",
                          block=BS, rows=T)
    # a stage behind an operator reads what it wrote
    p.fused("total", (1,), B, [(ir.reindex(plan.starts, (B,), [(((1, 0),), 1)]), (STREAM,))], C.plain(ir.M_MAX), ir.F32)
    g.update("held", "plan.held")
    free = np.arange(F)[::-1]
    ins = {n: dev.from_values(v, ir.U32) for n, v in (("past", [0] * B), ("new", [0] * B), ("free", free))}
    m = g.compile_for(dev).instantiate(ins)
    past, h, tables = [0] * B, [0] * (B + 1), np.zeros((B, M), np.int64)
    for new in ([3, 0, 9], [4, 1, 1], [1, 1, 1], [9, 9, 9]):
        m.write("past", past)
        m.write("new", new)
        m.step()
        starts, slots, positions, h, tables = ref.block_tables(past, new, h, free, tables, BS, T)
        assert m.read("plan.slots").astype(np.int64)[:starts[-1]].tolist() == [s if s != NONE else int(np.float64(np.uint32(NONE))) for s in slots]
        assert m.read("held").tolist() == h and m.read("total").tolist() == [starts[-1]]
        past = [a + b for a, b in zip(past, new)]
