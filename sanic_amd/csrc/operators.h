// Operator stages (SANIC_STAGE_OPERATOR): their checks and lowerings. Each has one file of kernels
// (op_tables.cpp: block tables and the cache write, op_attention.cpp, op_verify.cpp).
#pragma once
#include <string>
#include <vector>

#include "emit.h"

namespace sanic {

// A leaf that is an affine view of one buffer: element (c0, c1, ...) stands at base + Σ stride·c.
struct OperandView {
    int buffer = -1, dtype = -1;
    int64_t base = 0;
    std::vector<int64_t> stride, extent;
};
bool operand_view(const sanic_program_desc* d, int node, OperandView& out);

void validate_operator(const sanic_program_desc* d, int si);
// Program buffers that operator stage `st` writes, its output buffer first; those it reads.
std::vector<int> operator_writes(const sanic_program_desc* d, const sanic_stage& st);
std::vector<int> operator_reads(const sanic_program_desc* d, const sanic_stage& st);

LoweredStage lower_operator(const sanic_program_desc* d, int si, int64_t& scratch);
LoweredStage lower_block_tables(const sanic_program_desc* d, const sanic_stage& st);
LoweredStage lower_cache_write(const sanic_program_desc* d, const sanic_stage& st);
LoweredStage lower_paged_attn(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch);
LoweredStage lower_verify_drafts(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch);

// "constexpr long long NAME = value;" for a generated source
std::string constant(const char* name, int64_t v);
// Kernel functions: one element of a float type as f32 (sanic_get<code>), f32 rounded to one
// (sanic_put<code>), and the storage types by their code (sanic_elem<code>::T).
extern const char* kElement;

}  // namespace sanic
