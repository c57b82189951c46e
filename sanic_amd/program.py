"""Schedules as data: buffers, stages and the program descriptor handed across the C ABI.

Restates the backend's input contract: `Stage::{Fused, Elementwise/Gather}` and `Schedule`
(/root/reference/src/partition.rs:44-127), `FoldSched` (/root/reference/src/plan.rs:434-476),
and `Graph::{state, input, update, output}` (/root/reference/src/graph.rs:51-125). A `Program`
is what the reference's partitioner produces for one graph: an ordered list of stages whose
leaves are node trees over program buffers.
"""
from __future__ import annotations

import ctypes
import math
from collections import namedtuple
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from . import abi, ir
from .carrier import Carrier, ExprTable

INPUT, STATE, OUTPUT, SCRATCH = range(4)
STREAM, BCAST = -1, -2

# operators (include/sanic_hip.h SANIC_OPR_*) and the whole number that stands for no block, slot
# or token
BLOCK_TABLES, CACHE_WRITE, PAGED_ATTN, VERIFY_DRAFTS = 1, 2, 3, 4
NONE = 0xFFFFFFFF

BlockTables = namedtuple("BlockTables", "starts slots positions held tables")
Verified = namedtuple("Verified", "tokens accepted")


@dataclass
class Sched:
    """FoldSched re-derived for wave64: `lane_stream` lanes split the stream, `waves`
    wavefronts per workgroup, `chunk` contiguous elements per lane, `split` workgroups per
    output point merged by the carrier's combine (split-K / Flash-Decoding). A stage built
    without a Sched carries `waves = 0` (not lane_stream, split 1): the backend prices its
    candidate schedules and picks one (plan.rs:604-850); `Sched()` itself is the scalar form."""
    lane_stream: bool = False
    waves: int = 1
    chunk: int = 1
    split: int = 1
    variant: int = 0          # tiling variant of the kernel that lowers the stage (the tuner's)


@dataclass
class BufferDecl:
    name: str
    role: int
    dtype: int
    shape: Tuple[int, ...]
    index: int

    @property
    def nbytes(self) -> int:
        return ir.dtype_bytes(self.dtype, int(np.prod(self.shape)) if self.shape else 1)


@dataclass
class Stage:
    kind: int                       # 0 fused, 1 pointwise, 2 operator
    name: str
    out: BufferDecl
    grid: Tuple[int, ...]
    stream: int = 0
    leaves: List[Tuple[ir.Node, Tuple[int, ...]]] = field(default_factory=list)
    carrier: Optional[Carrier] = None
    epilogue: Optional[ir.Node] = None
    sched: Sched = field(default_factory=Sched)
    value: Optional[ir.Node] = None
    where: Optional[ir.Node] = None
    op: int = 0                     # operator: which one


class Program:
    """A schedule for the backend: declared buffers plus ordered stages."""

    def __init__(self):
        self.buffers: List[BufferDecl] = []
        self.by_name: Dict[str, BufferDecl] = {}
        self.stages: List[Stage] = []

    # ── buffers ──
    def _decl(self, name, role, shape, dtype) -> BufferDecl:
        if name in self.by_name:
            raise ValueError(f"buffer {name!r} declared twice")
        b = BufferDecl(name, role, dtype, tuple(int(s) for s in shape), len(self.buffers))
        self.buffers.append(b)
        self.by_name[name] = b
        return b

    def node(self, name: str) -> ir.Node:
        """A fresh Input node reading buffer `name`."""
        b = self.by_name[name]
        return ir.input_(name, b.shape, b.dtype)

    def input(self, name: str, shape, dtype=ir.F32) -> ir.Node:
        self._decl(name, INPUT, shape, dtype)
        return self.node(name)

    def state(self, name: str, shape, dtype=ir.F32) -> ir.Node:
        """Graph::state (graph.rs:51-80): caller-bound, rewritten in place by a stage."""
        self._decl(name, STATE, shape, dtype)
        return self.node(name)

    # ── stages ──
    def fused(self, name: str, grid, stream: int, leaves, carrier: Carrier, out_dtype=ir.F32,
              epilogue: Optional[ir.Node] = None, sched: Optional[Sched] = None,
              role: int = OUTPUT) -> ir.Node:
        """Stage::Fused: fold `carrier` over `stream` for every point of `grid`. `leaves` are
        (node, binding) pairs; binding[j] names the grid dim, STREAM or BCAST for leaf dim j."""
        if len(leaves) > abi.MAX_LEAVES:
            raise ValueError("too many leaves")
        out = self._decl(name, role, grid, out_dtype)
        lv = [(n, tuple(b)) for n, b in leaves]
        self.stages.append(Stage(0, name, out, tuple(grid), int(stream), lv, carrier, epilogue,
                                 sched or Sched(waves=0)))
        return self.node(name)

    def pointwise(self, name: str, value: ir.Node, out_dtype=ir.F32, grid=None,
                  where: Optional[ir.Node] = None, into: Optional[str] = None,
                  role: int = OUTPUT) -> ir.Node:
        """Stage::Elementwise / Gather. With `into`, the stage rewrites an existing (state)
        buffer in place and stores only where `where` is nonzero (emit_metal.rs:1103-1178)."""
        grid = tuple(grid if grid is not None else value.shape)
        if into is not None:
            out = self.by_name[into]
            if tuple(out.shape) != grid:
                raise ValueError("in-place grid must equal the state's shape")
        else:
            out = self._decl(name, role, grid, out_dtype)
        self.stages.append(Stage(1, name, out, grid, value=value, where=where))
        return self.node(out.name)

    # ── operators over a ragged batch and a paged cache (include/sanic_hip.h SANIC_STAGE_OPERATOR) ──
    def _operator(self, op: int, name: str, out: BufferDecl, operands, size: int = 0):
        leaves = [(n, ()) for n in operands]
        self.stages.append(Stage(2, name, out, tuple(out.shape), int(size), leaves, op=op))

    def _operand(self, x) -> ir.Node:
        return self.node(x) if isinstance(x, str) else x

    def block_tables(self, name: str, past, new, held, free, tables, block: int, rows: int, role: int = OUTPUT) -> BlockTables:
        """Where a step's new tokens go, from the requests' lengths. Request b holds `past[b]`
        tokens and brings `new[b]` (u32 [B]); `held` (u32 [B + 1]) counts the blocks that stand in
        each line of the state `tables` (u32 [B, M]) and, last, those taken from the list `free`
        (u32 [F]). Each request, in order, gets the blocks of `block` tokens that its new positions
        need, while the table's line and the list last; only those entries of `tables` are written.

        Declares `<name>.starts` [B + 1] (request b has the rows from starts[b] to starts[b + 1]; cut
        at `rows`), `<name>.slots` and `<name>.positions` [rows] (slot = block·block size + offset,
        NONE where no block is left, where the block is NONE and where the slot would pass 32 bits;
        rows behind the last request are left as they were) and
        `<name>.held` [B + 1], `held` for the next step. Calling it again with the same inputs
        writes the same results. A request whose tokens were taken back (rejected drafts) keeps its
        blocks: `past` may fall, `held` stays."""
        past, new, held, free, tables = (self._operand(x) for x in (past, new, held, free, tables))
        B = past.shape[0]
        starts = self._decl(f"{name}.starts", role, (B + 1,), ir.U32)
        slots = self._decl(f"{name}.slots", role, (rows,), ir.U32)
        positions = self._decl(f"{name}.positions", role, (rows,), ir.U32)
        after = self._decl(f"{name}.held", role, (B + 1,), ir.U32)
        self._operator(BLOCK_TABLES, name, starts,
                       [past, new, held, free, tables, self.node(slots.name), self.node(positions.name), self.node(after.name)], block)
        return BlockTables(*(self.node(b.name) for b in (starts, slots, positions, after)), tables)

    def cache_write(self, name: str, k, v, slots, starts, k_cache, v_cache):
        """Write the step's rows k and v [T, NKV, HD] into the paged caches (states
        [NB, NKV, BS, HD], or a view of one with these dims) at their slots, converted to the cache's
        type with one rounding. Rows behind the last request and slots past the pool (NONE among
        them) write nothing; slots of one step differ from each other. Returns the cache nodes."""
        k, v, slots, starts, kc, vc = (self._operand(x) for x in (k, v, slots, starts, k_cache, v_cache))
        src = kc
        while src.inputs:
            src = src.inputs[0]
        self._operator(CACHE_WRITE, name, self.by_name[src.name], [k, v, slots, starts, kc, vc])
        return kc, vc

    def paged_attention(self, name: str, q, k_cache, v_cache, tables, starts, past, scale: Optional[float] = None,
                        window: int = 0, out_dtype=ir.BF16, role: int = OUTPUT) -> ir.Node:
        """Causal attention of a step's rows q [T, NH, HD] over the paged caches
        [NB, NKV, BS, HD], which hold the step's own rows too: request b's row i stands at
        past[b] + i and sees the keys up to there, with `window` > 0 the last `window` of them. Query
        head h reads key head h // (NH // NKV). A row that sees no key is 0; rows behind the last
        request are left as they were, and so are all rows where `starts` falls. `scale` defaults to
        1/√HD.

        With 16-bit q and caches, `out_dtype` chooses the bits of a softmax weight: F32 keeps 22 or
        more in every row; a 16-bit type 16 or more where a request brings up to 32 rows times
        NH // NKV, and for longer chunks one rounding of each weight to the caches' type (RMS error
        against 64 bits in bf16 2.3e-3, where the output's own rounding makes 1.7e-3)."""
        q, kc, vc, tables, starts, past = (self._operand(x) for x in (q, k_cache, v_cache, tables, starts, past))
        out = self._decl(name, role, q.shape, out_dtype)
        scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
        self._operator(PAGED_ATTN, name, out, [q, kc, vc, tables, starts, past, ir.const(scale)], window)
        return self.node(name)

    def verify_drafts(self, name: str, p, q, tokens, starts, u, draw, role: int = OUTPUT) -> Verified:
        """Accept or refuse drafted tokens so that what comes out is distributed as the target's own
        samples. tokens[r + 1] (u32 [T]) is the draft behind row r of the same request, p [T, V] the
        target's probabilities at each row and q [T, V] those the draft was drawn from (None: it was
        certain, as from a lookup). Drafts are accepted in order while u[r]·q < p (u f32 [T], uniform
        in [0, 1)); then one more token is drawn by draw[b] (f32 [B], uniform in [0, 1)): from
        max(p − q, 0) where a draft was refused, from p behind the last one.

        Declares `<name>.tokens` [T] (a request's accepted drafts, the drawn token, then NONE; rows
        behind the last request are left as they were) and `<name>.accepted` [B]."""
        p, tokens, starts, u, draw = (self._operand(x) for x in (p, tokens, starts, u, draw))
        out = self._decl(f"{name}.tokens", role, tokens.shape, ir.U32)
        accepted = self._decl(f"{name}.accepted", role, draw.shape, ir.U32)
        self._operator(VERIFY_DRAFTS, name, out, [p, None if q is None else self._operand(q), tokens, u, draw, starts, self.node(accepted.name)])
        return Verified(self.node(out.name), self.node(accepted.name))

    def repeat_stage(self, i: int, copies: int, fresh_inputs: bool = False) -> List[str]:
        """Append `copies` more instances of stage `i`, each writing its own output buffer
        (for timing one kernel as back-to-back launches inside one captured graph). With
        `fresh_inputs` every copy reads its own copies of the stage's INPUT buffers
        (`<name>.copy<r>`), so back-to-back launches do not find each other's inputs in cache."""
        import copy as _copy
        st = self.stages[i]
        if st.kind == 2 and st.op != PAGED_ATTN:
            raise ValueError("an operator with several results is not repeated")
        names = []
        for r in range(copies):
            name = f"{st.out.name}.copy{r}"
            out = self._decl(name, OUTPUT, st.out.shape, st.out.dtype)
            dup = _copy.copy(st)
            dup.out = out
            dup.name = name
            if fresh_inputs:
                memo: Dict[int, ir.Node] = {}

                def ren(n: ir.Node) -> ir.Node:
                    if id(n) in memo:
                        return memo[id(n)]
                    if n.kind == ir.INPUT and self.by_name[n.name].role == INPUT:
                        cn = f"{n.name}.copy{r}"
                        if cn not in self.by_name:
                            b = self.by_name[n.name]
                            self._decl(cn, INPUT, b.shape, b.dtype)
                        m = _copy.copy(n)
                        m.name = cn
                    elif n.inputs:
                        m = _copy.copy(n)
                        m.inputs = tuple(ren(c) for c in n.inputs)
                    else:
                        m = n
                    memo[id(n)] = m
                    return m
                if st.kind in (0, 2):
                    dup.leaves = [(ren(nd), b) for nd, b in st.leaves]
                    dup.epilogue = ren(st.epilogue) if st.epilogue is not None else None
                else:
                    dup.value = ren(st.value)
                    dup.where = ren(st.where) if st.where is not None else None
            self.stages.append(dup)
            names.append(name)
        return names

    # ── serialization ──
    def pack(self):
        """Return (ProgramDesc, keepalive) for the C ABI."""
        nt = ir.NodeTable(lambda n: self.by_name[n.name].index)
        et = ExprTable()
        stages = np.zeros(len(self.stages), dtype=abi.STAGE_DT)
        for i, s in enumerate(self.stages):
            r = stages[i]
            r["kind"] = s.kind
            r["out_buffer"] = s.out.index
            r["out_dtype"] = s.out.dtype
            r["rank"] = len(s.grid)
            r["grid"] = list(s.grid) + [0] * (abi.MAX_RANK - len(s.grid))
            r["epilogue"] = -1
            r["value"] = -1
            r["where"] = -1
            if s.kind == 2:
                r["op"] = s.op
                r["stream"] = s.stream
                r["n_leaves"] = len(s.leaves)
                r["leaf"] = [-1 if n is None else nt.add(n) for n, _ in s.leaves] + [-1] * (abi.MAX_LEAVES - len(s.leaves))
                r["bind"] = -3
            elif s.kind == 0:
                r["stream"] = s.stream
                r["n_leaves"] = len(s.leaves)
                leaf = [-1] * abi.MAX_LEAVES
                bind = np.full((abi.MAX_LEAVES, abi.MAX_RANK), -3, dtype=np.int32)
                for l, (node, b) in enumerate(s.leaves):
                    leaf[l] = nt.add(node)
                    if len(b) != node.rank:
                        raise ValueError(f"stage {s.name}: leaf {l} binding rank")
                    bind[l, :len(b)] = b
                r["leaf"] = leaf
                r["bind"] = bind
                c = s.carrier
                car = r["carrier"]
                car["slots"] = c.slots
                for k in range(c.slots):
                    car["kind"][k]["kind"] = c.kinds[k].kind
                    car["kind"][k]["monoid"] = c.kinds[k].monoid
                    car["kind"][k]["ref_slot"] = c.kinds[k].ref_slot
                    car["kind"][k]["ties"] = c.kinds[k].ties
                    car["identity"][k] = c.identity[k]
                    car["into"][k] = et.add(c.into[k])
                    car["combine"][k] = et.add(c.combine[k])
                car["project"] = et.add(c.project)
                r["carrier"] = car
                if s.epilogue is not None:
                    r["epilogue"] = nt.add(s.epilogue)
                r["sched"]["lane_stream"] = int(s.sched.lane_stream)
                r["sched"]["waves"] = s.sched.waves
                r["sched"]["chunk"] = s.sched.chunk
                r["sched"]["split"] = s.sched.split
                r["sched"]["variant"] = s.sched.variant
            else:
                r["value"] = nt.add(s.value)
                if s.where is not None:
                    r["where"] = nt.add(s.where)
        nodes = nt.pack()
        exprs = et.pack()
        reindex = np.array(nt.reindex or [0], dtype=np.int64)
        bufs = np.zeros(len(self.buffers), dtype=abi.BUFFER_DT)
        for i, b in enumerate(self.buffers):
            bufs[i]["role"] = b.role
            bufs[i]["dtype"] = b.dtype
            bufs[i]["scale"] = ir.dtype_scale(b.dtype)
            bufs[i]["rank"] = len(b.shape)
            bufs[i]["shape"] = list(b.shape) + [0] * (abi.MAX_RANK - len(b.shape))
        keep = [nodes, exprs, reindex, bufs, stages]
        desc = abi.ProgramDesc(
            len(nodes), nodes.ctypes.data, len(exprs), exprs.ctypes.data,
            len(nt.reindex), reindex.ctypes.data, len(bufs), bufs.ctypes.data,
            len(stages), stages.ctypes.data)
        return desc, keep

    def emit(self, stage: int) -> Tuple[str, str]:
        """(kernel kind, HIP source) of one stage — no GPU needed."""
        desc, keep = self.pack()
        kind = ctypes.create_string_buffer(256)
        cap = 1 << 22
        src = ctypes.create_string_buffer(cap)
        abi.check(abi.lib().sanic_hip_emit_source(ctypes.byref(desc), stage, kind, 256, src, cap))
        return kind.value.decode(), src.value.decode()

    def stage_variants(self, stage: int = -1):
        """Tiling variants the kernel lowering `stage` offers (0: folded into another launch);
        with stage = -1 the list for every stage, from one lowering."""
        desc, keep = self.pack()
        n = (ctypes.c_int * max(1, len(self.stages)))()
        abi.check(abi.lib().sanic_hip_stage_variants(ctypes.byref(desc), stage, n))
        return list(n[:len(self.stages)]) if stage == -1 else n[0]

    def with_variants(self, variants: Dict[int, int]) -> "Program":
        """A copy whose stages carry the given tiling variants (stage index -> variant)."""
        import copy as _copy
        import dataclasses
        p = _copy.copy(self)
        p.stages = list(self.stages)
        for i, v in variants.items():
            st = _copy.copy(p.stages[i])
            st.sched = dataclasses.replace(st.sched or Sched(), variant=int(v))
            p.stages[i] = st
        return p

    def precompile(self):
        desc, keep = self.pack()
        abi.check(abi.lib().sanic_hip_precompile(ctypes.byref(desc)))
