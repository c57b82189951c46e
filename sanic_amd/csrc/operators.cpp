// Operator stages: operand checks and what they share. The operands and their meaning are stated at
// SANIC_STAGE_OPERATOR in include/sanic_hip.h.
#include "operators.h"

#include <algorithm>

#include "skeletons.h"

namespace sanic {

const char* kElement = R"SRC(
// storage codes: 1 f32, 2 f16, 3 bf16
template <int DT> struct sanic_elem;
template <> struct sanic_elem<1> { typedef float T; };
template <> struct sanic_elem<2> { typedef _Float16 T; };
template <> struct sanic_elem<3> { typedef unsigned short T; };
template <int DT> __device__ __forceinline__ float sanic_get(typename sanic_elem<DT>::T v) {
  if constexpr (DT == 3) return sanic_bf16(v);
  else return (float)v;
}
// one rounding to the storage type, ties to even (float to _Float16 rounds so as well)
template <int DT> __device__ __forceinline__ typename sanic_elem<DT>::T sanic_put(float v) {
  if constexpr (DT == 3) return sanic_to_bf16(v);
  else return (typename sanic_elem<DT>::T)v;
}
)SRC";

std::string constant(const char* name, int64_t v) {
    return std::string("constexpr long long ") + name + " = " + std::to_string(v) + "LL;\n";
}

bool operand_view(const sanic_program_desc* d, int node, OperandView& out) {
    const sanic_node& n = d->nodes[node];
    std::vector<Sym> c;
    std::vector<int64_t> ext;
    for (int j = 0; j < n.rank; j++) {
        c.push_back(Sym::var(j));
        ext.push_back(n.shape[j]);
    }
    Access a;
    if (!sym_access(d, node, c, ext, a)) return false;
    out.buffer = a.buffer;
    out.dtype = a.dtype;
    out.base = a.addr.c0;
    out.stride.assign(n.rank, 0);
    out.extent = ext;
    for (auto& t : a.addr.terms) {
        if (ext[t.var] == 1) continue;
        if (t.div != 1 || (t.mod && t.mod < ext[t.var])) return false;
        out.stride[t.var] += t.coef;
    }
    return true;
}

static bool is_float(int dt) { return dt == SANIC_F32 || dt == SANIC_F16 || dt == SANIC_BF16; }

// leaves of each operator that it writes beside its output buffer
static std::vector<int> written_leaves(int op) {
    switch (op) {
    case SANIC_OPR_BLOCK_TABLES: return {4, 5, 6, 7};
    case SANIC_OPR_CACHE_WRITE: return {4, 5};
    case SANIC_OPR_VERIFY_DRAFTS: return {6};
    default: return {};
    }
}

static int buffer_of(const sanic_program_desc* d, int node) {
    while (d->nodes[node].kind == SANIC_NODE_REINDEX || d->nodes[node].kind == SANIC_NODE_VIEW) node = d->nodes[node].in[0];
    return d->nodes[node].kind == SANIC_NODE_INPUT ? d->nodes[node].buffer : -1;
}

std::vector<int> operator_writes(const sanic_program_desc* d, const sanic_stage& st) {
    std::vector<int> out{st.out_buffer};
    for (int l : written_leaves(st.op)) {
        const int b = buffer_of(d, st.leaf[l]);
        if (std::find(out.begin(), out.end(), b) == out.end()) out.push_back(b);
    }
    return out;
}

std::vector<int> operator_reads(const sanic_program_desc* d, const sanic_stage& st) {
    const std::vector<int> w = operator_writes(d, st);
    std::vector<int> out;
    for (int l = 0; l < st.n_leaves; l++) {
        const int b = st.leaf[l] < 0 ? -1 : buffer_of(d, st.leaf[l]);
        if (b >= 0 && std::find(w.begin(), w.end(), b) == w.end()) out.push_back(b);
    }
    return out;
}

void validate_operator(const sanic_program_desc* d, int si) {
    const sanic_stage& st = d->stages[si];
    static const char* names[] = {"", "block_tables", "cache_write", "paged_attention", "verify_drafts"};
    static const int leaves[] = {0, 8, 6, 7, 7};
    if (st.op < SANIC_OPR_BLOCK_TABLES || st.op > SANIC_OPR_VERIFY_DRAFTS)
        fail(SANIC_ERR_COMPILE, "stage " + std::to_string(si) + ": unknown operator");
    auto bad = [&](const std::string& m, int code = SANIC_ERR_COMPILE) {
        fail(code, "stage " + std::to_string(si) + " (" + names[st.op] + "): " + m);
    };
    if (st.n_leaves != leaves[st.op]) bad("takes " + std::to_string(leaves[st.op]) + " leaves");
    for (int l = 0; l < st.n_leaves; l++) {
        const bool optional = st.op == SANIC_OPR_VERIFY_DRAFTS && l == 1;
        if (st.leaf[l] >= d->n_nodes || st.leaf[l] < (optional ? -1 : 0)) bad("leaf node");
    }
    auto node = [&](int l) -> const sanic_node& { return d->nodes[st.leaf[l]]; };
    auto rank = [&](int l, int r, const char* what) {
        if (node(l).rank != r) bad(std::string(what) + " has rank " + std::to_string(node(l).rank) + ", not " + std::to_string(r), SANIC_ERR_SHAPE);
    };
    auto extent = [&](int l, int j, int64_t want, const char* what) {
        if (node(l).shape[j] != want)
            bad(std::string(what) + " has extent " + std::to_string(node(l).shape[j]) + " along dim " + std::to_string(j) + ", not " + std::to_string(want),
                SANIC_ERR_SHAPE);
    };
    // a whole buffer of whole numbers (or, with dt, of that type)
    auto plain = [&](int l, const char* what, int dt = SANIC_U32) {
        if (node(l).kind != SANIC_NODE_INPUT) bad(std::string(what) + " is not a buffer");
        if (node(l).dtype != dt) bad(std::string(what) + (dt == SANIC_U32 ? " is not u32" : " is not f32"), SANIC_ERR_DTYPE);
    };
    auto floats = [&](int l, const char* what) {
        OperandView v;
        if (!operand_view(d, st.leaf[l], v)) bad(std::string(what) + " is not an affine view of a buffer");
        if (!is_float(v.dtype)) bad(std::string(what) + " is not f32, f16 or bf16", SANIC_ERR_DTYPE);
        return v;
    };
    auto written = [&](int l, const char* what, bool state) {
        if (buffer_of(d, st.leaf[l]) < 0) bad(std::string(what) + " is not a buffer");
        const int role = d->buffers[buffer_of(d, st.leaf[l])].role;
        if (state ? role != SANIC_BUF_STATE : role == SANIC_BUF_INPUT) bad(std::string(what) + (state ? " is not a state" : " is an input buffer"));
    };
    // a view that is written covers its buffer one to one (no repeated and no skipped element)
    auto whole = [&](const OperandView& v, const char* what) {
        int64_t n = 1, all = 1;
        std::vector<std::pair<int64_t, int64_t>> o;
        for (size_t j = 0; j < v.extent.size(); j++)
            if (v.extent[j] > 1) o.push_back({v.stride[j], v.extent[j]});
        std::sort(o.begin(), o.end());
        bool dense = v.base == 0;
        for (auto& p : o) {
            dense = dense && p.first == n;
            n *= p.second;
        }
        const sanic_buffer_desc& b = d->buffers[v.buffer];
        for (int j = 0; j < b.rank; j++) all *= b.shape[j];
        if (!dense || n != all) bad(std::string(what) + " is not its whole buffer in some order of dims");
    };
    const sanic_buffer_desc& out = d->buffers[st.out_buffer];
    const auto limit = [&](int64_t v, int64_t most, const char* what) {
        if (v > most) bad(std::string(what) + " is " + std::to_string(v) + ", at most " + std::to_string(most) + " are supported", SANIC_ERR_SHAPE);
    };
    const int64_t kWord = 0xFFFFFFFFLL;
    if (st.op == SANIC_OPR_BLOCK_TABLES) {
        static const char* what[] = {"past", "new", "held", "free", "tables", "slots", "positions", "held_next"};
        for (int l = 0; l < 8; l++) {
            plain(l, what[l]);
            rank(l, l == 4 ? 2 : 1, what[l]);
        }
        const int64_t B = node(0).shape[0], T = node(5).shape[0];
        extent(1, 0, B, "new"), extent(2, 0, B + 1, "held"), extent(4, 0, B, "tables"), extent(6, 0, T, "positions"), extent(7, 0, B + 1, "held_next");
        written(4, "tables", true), written(5, "slots", false), written(6, "positions", false), written(7, "held_next", false);
        if (st.out_dtype != SANIC_U32 || out.rank != 1 || out.shape[0] != B + 1) bad("starts is not u32 [B + 1]", SANIC_ERR_SHAPE);
        if (st.stream < 1 || st.stream > (1 << 30)) bad("block size", SANIC_ERR_SHAPE);
        limit(B, 8192, "the number of requests");
        limit(T, int64_t(1) << 30, "the number of rows"), limit(node(3).shape[0], int64_t(1) << 30, "the free list");
        limit(B * node(4).shape[1], int64_t(1) << 40, "the block table");
    } else if (st.op == SANIC_OPR_CACHE_WRITE) {
        rank(0, 3, "k"), rank(1, 3, "v"), rank(2, 1, "slots"), rank(3, 1, "starts"), rank(4, 4, "the key cache"), rank(5, 4, "the value cache");
        plain(2, "slots"), plain(3, "starts");
        const int64_t T = node(0).shape[0], NKV = node(0).shape[1], HD = node(0).shape[2];
        extent(1, 0, T, "v"), extent(1, 1, NKV, "v"), extent(1, 2, HD, "v"), extent(2, 0, T, "slots");
        for (int l = 4; l < 6; l++) {
            extent(l, 0, node(4).shape[0], "the cache"), extent(l, 1, NKV, "the cache"), extent(l, 2, node(4).shape[2], "the cache");
            extent(l, 3, HD, "the cache");
            written(l, "the cache", true);
            whole(floats(l, "the cache"), "the cache");
        }
        floats(0, "k"), floats(1, "v");
        if (buffer_of(d, st.leaf[4]) == buffer_of(d, st.leaf[5])) bad("keys and values share a buffer");
        if (buffer_of(d, st.leaf[4]) != st.out_buffer) bad("the output is not the key cache");
        limit(T, int64_t(1) << 30, "the number of rows"), limit(node(4).shape[0] * node(4).shape[2], kWord, "the number of slots");
        limit(NKV * HD, int64_t(1) << 24, "a token's row");
    } else if (st.op == SANIC_OPR_PAGED_ATTN) {
        rank(0, 3, "q"), rank(1, 4, "the key cache"), rank(2, 4, "the value cache"), rank(3, 2, "tables"), rank(4, 1, "starts"), rank(5, 1, "past");
        plain(3, "tables"), plain(4, "starts"), plain(5, "past");
        const int64_t T = node(0).shape[0], NH = node(0).shape[1], HD = node(0).shape[2], B = node(3).shape[0];
        const int64_t NKV = node(1).shape[1];
        extent(1, 3, HD, "the key cache");
        for (int j = 0; j < 4; j++) extent(2, j, node(1).shape[j], "the value cache");
        extent(4, 0, B + 1, "starts"), extent(5, 0, B, "past");
        if (NH % NKV) bad(std::to_string(NH) + " query heads over " + std::to_string(NKV) + " key heads", SANIC_ERR_SHAPE);
        const OperandView q = floats(0, "q"), k = floats(1, "the key cache"), v = floats(2, "the value cache");
        if (k.dtype != v.dtype) bad("keys and values differ in type", SANIC_ERR_DTYPE);
        (void)q;
        if (node(6).kind != SANIC_NODE_CONST) bad("the scale is not a constant");
        if (!is_float(st.out_dtype) || out.rank != 3 || out.shape[0] != T || out.shape[1] != NH || out.shape[2] != HD)
            bad("the output is not a float buffer of q's shape", SANIC_ERR_SHAPE);
        if (st.stream < 0) bad("window", SANIC_ERR_SHAPE);
        limit(B, 8192, "the number of requests"), limit(HD, 512, "the head size"), limit(T * NH, int64_t(1) << 26, "the number of rows times heads");
        limit(node(1).shape[0] * node(1).shape[2], kWord, "the number of slots");
        limit(node(3).shape[1] * node(1).shape[2], int64_t(1) << 30, "a request's tokens");
    } else {
        rank(0, 2, "p"), rank(2, 1, "tokens"), rank(3, 1, "u"), rank(4, 1, "draw"), rank(5, 1, "starts"), rank(6, 1, "accepted");
        plain(2, "tokens"), plain(3, "u", SANIC_F32), plain(4, "draw", SANIC_F32), plain(5, "starts"), plain(6, "accepted");
        const int64_t T = node(0).shape[0], V = node(0).shape[1], B = node(4).shape[0];
        floats(0, "p");
        if (st.leaf[1] >= 0) {
            rank(1, 2, "q"), extent(1, 0, T, "q"), extent(1, 1, V, "q");
            floats(1, "q");
        }
        extent(2, 0, T, "tokens"), extent(3, 0, T, "u"), extent(5, 0, B + 1, "starts"), extent(6, 0, B, "accepted");
        written(6, "accepted", false);
        if (st.out_dtype != SANIC_U32 || out.rank != 1 || out.shape[0] != T) bad("the tokens are not u32 [T]", SANIC_ERR_SHAPE);
        limit(B, 65536, "the number of requests"), limit(T, int64_t(1) << 26, "the number of rows"), limit(V, int64_t(1) << 30, "the vocabulary");
    }
    const std::vector<int> w = operator_writes(d, st);
    for (int l = 0; l < st.n_leaves; l++) {
        const auto wl = written_leaves(st.op);
        if (st.leaf[l] < 0 || std::find(wl.begin(), wl.end(), l) != wl.end()) continue;
        const int b = buffer_of(d, st.leaf[l]);
        if (b >= 0 && std::find(w.begin(), w.end(), b) != w.end()) bad("reads a buffer that it writes");
    }
    if (w.size() != written_leaves(st.op).size() + (st.op == SANIC_OPR_CACHE_WRITE ? 0 : 1)) bad("two results share a buffer");
}

LoweredStage lower_operator(const sanic_program_desc* d, int si, int64_t& scratch) {
    const sanic_stage& st = d->stages[si];
    switch (st.op) {
    case SANIC_OPR_BLOCK_TABLES: return lower_block_tables(d, st);
    case SANIC_OPR_CACHE_WRITE: return lower_cache_write(d, st);
    case SANIC_OPR_PAGED_ATTN: return lower_paged_attn(d, st, scratch);
    default: return lower_verify_drafts(d, st, scratch);
    }
}

}  // namespace sanic
