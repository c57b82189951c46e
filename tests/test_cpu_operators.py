"""What the operators over ragged batches and paged caches refuse, on the CPU: shapes, types, roles
and views, each before a kernel is compiled; and that what they accept lowers onto their kernels."""
import re

import pytest

from sanic_amd import abi, configs, ir
from sanic_amd.abi import SanicError
from sanic_amd.program import INPUT, STATE, Program

ARG, COMPILE, SHAPE, DTYPE = 7, 1, 3, 4


def tables(B=3, F=9, M=4, T=5, block=16, **other):
    """other: a buffer's shape, or (shape, dtype), or for `state` False."""
    p = Program()

    def buf(name, shape, role=INPUT):
        o = other.get(name, shape)
        shape, dtype = o if isinstance(o[0], tuple) else (o, ir.U32)
        return (p.state if role == STATE else p.input)(name, shape, dtype)

    buf("tables", (B, M), STATE if other.get("state", True) else INPUT)
    p.block_tables("plan", buf("past", (B,)), buf("new", (B,)), buf("held", (B + 1,)), buf("free", (F,)), "tables", block=block, rows=T)
    return p


def write(T=5, NKV=2, HD=16, NB=4, BS=8, B=2, src=ir.F32, dst=ir.BF16, k=None, v=None, kc=None, vc=None, slots=None, starts=None):
    p = Program()
    names = {"k": (k, (T, NKV, HD), src), "v": (v, (T, NKV, HD), src), "slots": (slots, (T,), ir.U32), "starts": (starts, (B + 1,), ir.U32)}
    nodes = {n: p.input(n, *(o if o else (shape, dt))) for n, (o, shape, dt) in names.items()}
    for n, o in (("kc", kc), ("vc", vc)):
        nodes[n] = o(p) if callable(o) else p.state(n, *(o if o else ((NB, NKV, BS, HD), dst)))
    p.cache_write("write", *(nodes[n] for n in ("k", "v", "slots", "starts", "kc", "vc")))
    return p


def attn(T=5, NH=4, NKV=2, HD=64, NB=6, BS=16, B=2, M=3, dtype=ir.BF16, out=ir.BF16, window=0, scale=None, **other):
    p = Program()
    shapes = {"q": ((T, NH, HD), dtype), "kc": ((NB, NKV, BS, HD), dtype), "vc": ((NB, NKV, BS, HD), dtype), "tables": ((B, M), ir.U32),
              "starts": ((B + 1,), ir.U32), "past": ((B,), ir.U32)}
    nodes = [other[n](p) if callable(other.get(n)) else p.input(n, *other.get(n, s)) for n, s in shapes.items()]
    p.paged_attention("o", *nodes, scale=scale, window=window, out_dtype=out)
    return p


def verify(T=5, V=100, B=2, with_q=True, **other):
    p = Program()
    shapes = {"p": ((T, V), ir.F32), "q": ((T, V), ir.F32), "tokens": ((T,), ir.U32), "starts": ((B + 1,), ir.U32), "u": ((T,), ir.F32),
              "draw": ((B,), ir.F32)}
    nodes = [None if n == "q" and not with_q else p.input(n, *other.get(n, s)) for n, s in shapes.items()]
    p.verify_drafts("check", *nodes)
    return p


@pytest.mark.parametrize("build,kind", [
    (tables, "operator:block_tables"), (lambda: tables(B=1, F=1, M=1, T=1, block=1), "operator:block_tables"),
    (lambda: tables(B=8192), "operator:block_tables"),
    (write, "operator:cache_write"), (lambda: write(HD=7), "operator:cache_write[scalar]"), (lambda: write(src=ir.F16, dst=ir.F32), "operator:cache_write"),
    (attn, "operator:paged_attn"), (lambda: attn(HD=7, dtype=ir.F32, out=ir.F32), "operator:paged_attn[plain]"),
    (verify, "operator:verify_drafts"), (lambda: verify(with_q=False), "operator:verify_drafts"), (lambda: verify(V=1, B=1, T=1), "operator:verify_drafts"),
])
def test_accepted(build, kind):
    p = build()
    got, source = p.emit(0)
    assert got.startswith(kind) and "__global__" in source
    assert p.stage_variants(0) >= 1


REFUSED = {
    "tables: past not u32": (lambda: tables(past=((3,), ir.F32)), DTYPE),
    "tables: tables not u32": (lambda: tables(tables=((3, 4), ir.F32)), DTYPE),
    "tables: new of another length": (lambda: tables(new=(4,)), SHAPE),
    "tables: held without the list's count": (lambda: tables(held=(3,)), SHAPE),
    "tables: tables of another length": (lambda: tables(tables=(4, 4)), SHAPE),
    "tables: tables of rank 1": (lambda: tables(tables=(12,)), SHAPE),
    "tables: tables not a state": (lambda: tables(state=False), COMPILE),
    "tables: no block size": (lambda: tables(block=0), SHAPE),
    "tables: negative block size": (lambda: tables(block=-16), SHAPE),
    "tables: too many requests": (lambda: tables(B=8193), SHAPE),
    "write: q8 rows": (lambda: write(k=((5, 2, 16), ir.q8(0.5))), DTYPE),
    "write: u32 cache": (lambda: write(dst=ir.U32), DTYPE),
    "write: rows and cache of different heads": (lambda: write(k=((5, 3, 16), ir.F32)), SHAPE),
    "write: rows and cache of different sizes": (lambda: write(kc=((4, 2, 8, 32), ir.BF16)), SHAPE),
    "write: values of another length": (lambda: write(v=((6, 2, 16), ir.F32)), SHAPE),
    "write: pools of different sizes": (lambda: write(vc=((5, 2, 8, 16), ir.BF16)), SHAPE),
    "write: slots of another length": (lambda: write(slots=((6,), ir.U32)), SHAPE),
    "write: slots not u32": (lambda: write(slots=((5,), ir.F32)), DTYPE),
    "write: cache an input": (lambda: write(kc=lambda p: p.input("kc", (4, 2, 8, 16), ir.BF16)), COMPILE),
    "write: cache view that repeats heads": (
        lambda: write(vc=lambda p: ir.reindex(p.state("vc", (4, 1, 8, 16), ir.BF16), (4, 2, 8, 16), [(((1, 0),), 0), ((), 0), (((1, 2),), 0), (((1, 3),), 0)])), COMPILE),
    "write: cache view of a part": (
        lambda: write(vc=lambda p: ir.reindex(p.state("vc", (4, 3, 8, 16), ir.BF16), (4, 2, 8, 16), [(((1, i),), 0) for i in range(4)])), COMPILE),
    "write: k computed": (lambda: _computed_k(), COMPILE),
    "write: one buffer for keys and values": (lambda: _one_cache(), COMPILE),
    "attn: heads that do not divide": (lambda: attn(NH=5), SHAPE),
    "attn: cache of another head size": (lambda: attn(kc=((6, 2, 16, 32), ir.BF16)), SHAPE),
    "attn: values of another pool": (lambda: attn(vc=((7, 2, 16, 64), ir.BF16)), SHAPE),
    "attn: keys and values of different types": (lambda: attn(vc=((6, 2, 16, 64), ir.F16)), DTYPE),
    "attn: q8 cache": (lambda: attn(kc=((6, 2, 16, 64), ir.q8(0.1)), vc=((6, 2, 16, 64), ir.q8(0.1))), DTYPE),
    "attn: starts without the end": (lambda: attn(starts=((2,), ir.U32)), SHAPE),
    "attn: past of another length": (lambda: attn(past=((3,), ir.U32)), SHAPE),
    "attn: past not u32": (lambda: attn(past=((2,), ir.F32)), DTYPE),
    "attn: tables of rank 1": (lambda: attn(tables=((6,), ir.U32)), SHAPE),
    "attn: q of rank 2": (lambda: attn(q=((5, 256), ir.BF16)), SHAPE),
    "attn: u32 output": (lambda: attn(out=ir.U32), SHAPE),
    "attn: negative window": (lambda: attn(window=-1), SHAPE),
    "attn: head size": (lambda: attn(HD=513), SHAPE),
    "attn: q computed": (lambda: attn(q=lambda p: ir.map_(ir.ADD, p.input("q", (5, 4, 64), ir.BF16), ir.const(1.0))), COMPILE),
    "attn: too many requests": (lambda: attn(B=8193), SHAPE),
    "verify: vocabularies differ": (lambda: verify(q=((5, 99), ir.F32)), SHAPE),
    "verify: tokens not u32": (lambda: verify(tokens=((5,), ir.F32)), DTYPE),
    "verify: u of another length": (lambda: verify(u=((4,), ir.F32)), SHAPE),
    "verify: u not f32": (lambda: verify(u=((5,), ir.BF16)), DTYPE),
    "verify: starts of another length": (lambda: verify(starts=((2,), ir.U32)), SHAPE),
    "verify: p of rank 1": (lambda: verify(p=((500,), ir.F32)), SHAPE),
    "verify: u32 probabilities": (lambda: verify(p=((5, 100), ir.U32)), DTYPE),
}


@pytest.mark.parametrize("which", ["kc", "vc"])
def test_blocks_read_backwards_take_the_plain_kernel(which):
    """The matrix-core kernel adds a row's place in its block as an unsigned offset."""
    p = attn(**{which: lambda p: ir.flip(p.input(which, (6, 2, 16, 64), ir.BF16), 2)})
    assert p.emit(0)[0] == "operator:paged_attn[plain]"
    p = attn(**{which: lambda p: ir.flip(p.input(which, (6, 2, 16, 64), ir.BF16), 1)})
    assert p.emit(0)[0] == "operator:paged_attn[mfma]"


def _computed_k():
    p = Program()
    k = ir.map_(ir.MUL, p.input("k", (5, 2, 16)), ir.const(2.0))
    p.cache_write("write", k, p.input("v", (5, 2, 16)), p.input("slots", (5,), ir.U32), p.input("starts", (3,), ir.U32),
                  p.state("kc", (4, 2, 8, 16)), p.state("vc", (4, 2, 8, 16)))
    return p


def _one_cache():
    p = Program()
    c = p.state("kc", (4, 2, 8, 16))
    p.cache_write("write", p.input("k", (5, 2, 16)), p.input("v", (5, 2, 16)), p.input("slots", (5,), ir.U32), p.input("starts", (3,), ir.U32), c, "kc")
    return p


@pytest.mark.parametrize("case", REFUSED)
def test_refused(case):
    build, code = REFUSED[case]
    with pytest.raises(SanicError) as e:
        build().emit(0)
    assert e.value.code == code, str(e.value)
    assert "stage 0" in str(e.value)


def test_unknown_operator_and_leaf_counts_are_refused():
    for change in (dict(op=0), dict(op=9), dict(leaves=3)):
        p = attn()
        st = p.stages[0]
        st.op = change.get("op", st.op)
        st.leaves = st.leaves[:change.get("leaves", 8)]
        with pytest.raises(SanicError) as e:
            p.emit(0)
        assert e.value.code == COMPILE


def test_a_leaf_may_not_be_missing():
    p = attn()
    p.stages[0].leaves[1] = (None, ())
    with pytest.raises(SanicError):
        p.emit(0)


def test_several_results_are_not_repeated():
    with pytest.raises(ValueError):
        tables().repeat_stage(0, 2)
    p = attn()
    p.repeat_stage(0, 2, fresh_inputs=True)
    assert [p.emit(i)[0] for i in range(3)] == [p.emit(0)[0]] * 3 and "kc.copy1" in p.by_name


def test_the_record_keeps_its_size():
    """The operator's code stands in what was padding before the carrier."""
    assert abi.STAGE_DT.fields["op"][1] == abi.STAGE_DT.fields["bind"][1] + 4 * abi.MAX_LEAVES * abi.MAX_RANK
    assert abi.STAGE_DT.fields["carrier"][1] == abi.STAGE_DT.fields["op"][1] + 4
    want, got = abi.check_layouts()
    assert want == got


def test_programs_without_operators_say_so():
    p = configs.direct_attention()
    desc, keep = p.pack()
    assert int(keep[4][0]["op"]) == 0


@pytest.mark.parametrize("NKV,T,kind", [(8, 5, "mfma"), (1024, 5, "mfma"), (1024, 40, "plain"), (4096, 1, "plain")])
def test_many_key_heads_keep_to_the_static_scratch(NKV, T, kind):
    """Where two parts a key head would not fit the partials' room, the kernel without parts takes the call."""
    assert attn(NH=NKV, NKV=NKV, HD=128, T=T).emit(0)[0] == f"operator:paged_attn[{kind}]"


@pytest.mark.parametrize("T,HD,runs", [(64, 128, 64), (1024, 128, 64), (1536, 128, 60), (2048, 128, 40), (1024, 64, 96), (2048, 64, 96)])
def test_a_whole_step_keeps_its_runs_of_keys(T, HD, runs):
    """The rotated rows of a long step take part of the static scratch: the attention's partials get what
    is left of it, not a fixed small part. Runs a key head of requests of up to 16 packed rows."""
    p = configs.paged_step(T, 41, 32, 8, HD, 4096, 16, 512)
    i = next(i for i, st in enumerate(p.stages) if st.kind == 2 and st.op == 3)
    kind, source = p.emit(i)
    assert kind == "operator:paged_attn[mfma]"
    c = {m[1]: int(m[2]) for m in re.finditer(r"constexpr int (\w+) = (\d+);", source)}
    assert min(c["FEW_GROUPS"], c["DROWS"] // 32) >= runs
