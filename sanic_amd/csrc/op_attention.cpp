// Attention of a ragged batch's new rows over a paged cache.
//
// Row r of request b stands at position p = past[b] + r − starts[b] and sees the keys of positions
// lo ≤ j ≤ p (lo = max(0, p + 1 − window)), where j's block is in the pool:
//   s_j = scale · q·k_j,  m = max s,  o = Σ exp(s_j − m)·v_j / Σ exp(s_j − m)
#include <algorithm>
#include <cmath>

#include "operators.h"

namespace sanic {

// One wave per (row, head), keys 64 at a time, one per lane for the scores and one value dim per lane
// for the output; m, the sum and the output in f32 over one pass. For every type, head size and
// layout.
static const char* kPlain = R"SRC(
typedef sanic_elem<DQ>::T q_t;
typedef sanic_elem<DC>::T kv_t;
typedef sanic_elem<DO>::T o_t;
struct Args { const q_t* q; const kv_t *k, *v; const unsigned *tables, *starts, *past; o_t* o; };
constexpr int DV = (HD + 63) / 64;

extern "C" __global__ void __launch_bounds__(256) sanic_paged_attn(Args a) {
  __shared__ float q_of[4][HD];
  __shared__ float w_of[4][64];
  __shared__ unsigned page_of[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long item = (long long)blockIdx.x * 4 + wave;
  const long long r = item / NH;
  const int h = (int)(item % NH), g = h / REP;
  if (r >= T || r >= a.starts[B]) return;
  int b = 0, hi_b = B;   // the last request that starts at or before r
  while (hi_b - b > 1) {
    const int mid = (b + hi_b) >> 1;
    if (a.starts[mid] <= r) b = mid; else hi_b = mid;
  }
  if (r < a.starts[b] || r >= a.starts[b + 1]) return;
  const long long p = (long long)a.past[b] + (r - a.starts[b]);
  const long long end = p + 1 < M * BS ? p + 1 : M * BS;
  const long long lo = W && p + 1 > W ? p + 1 - W : 0;
  for (int e = lane; e < HD; e += 64) q_of[wave][e] = sanic_get<DQ>(a.q[QB + r * Q0 + h * Q1 + e * Q2]) * SCALE;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  float m = -__builtin_huge_valf(), sum = 0.0f, o[DV];
  for (int i = 0; i < DV; i++) o[i] = 0.0f;
  for (long long base = lo / 64 * 64; base < end; base += 64) {
    const long long j = base + lane;
    unsigned page = 0xFFFFFFFFu;
    if (j >= lo && j < end) page = a.tables[(long long)b * M + j / BS];
    const bool seen = page < NB;
    float s = -__builtin_huge_valf();
    if (seen) {
      const kv_t* k = a.k + (KB + page * K0 + g * K1 + j % BS * K2);
      float dot = 0.0f;
      for (int e = 0; e < HD; e++) dot = __builtin_fmaf(q_of[wave][e], sanic_get<DC>(k[e * K3]), dot);
      s = dot;
    }
    const float top = __builtin_fmaxf(m, sanic_wave_max(s));
    // nothing seen so far, or only scores of -inf (whose weights are 0): no reference to subtract
    const float ref = top == -__builtin_huge_valf() ? 0.0f : top;
    const float w = seen ? __expf(s - ref) : 0.0f, c = __expf(m - ref);
    m = top;
    sum = sum * c + sanic_wave_sum(w);
    for (int i = 0; i < DV; i++) o[i] *= c;
    w_of[wave][lane] = w;
    page_of[wave][lane] = page;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int x = 0; x < 64; x++) {
      const unsigned pg = page_of[wave][x];
      if (pg >= NB) continue;   // a masked place's value may be anything, NaN among it
      const kv_t* v = a.v + (VB + pg * V0 + g * V1 + (base + x) % BS * V2);
      const float wx = w_of[wave][x];
      for (int i = 0; i < DV; i++)
        if (lane + 64 * i < HD) o[i] = __builtin_fmaf(wx, sanic_get<DC>(v[(lane + 64 * i) * V3]), o[i]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  for (int i = 0; i < DV; i++)
    if (lane + 64 * i < HD) a.o[(r * NH + h) * HD + lane + 64 * i] = sanic_put<DO>(sum == 0.0f ? 0.0f : o[i] / sum);
}
)SRC";

LoweredStage lower_paged_attn(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch) {
    (void)scratch;
    OperandView q, k, v;
    operand_view(d, st.leaf[0], q), operand_view(d, st.leaf[1], k), operand_view(d, st.leaf[2], v);
    const int64_t T = q.extent[0], NH = q.extent[1], HD = q.extent[2], NB = k.extent[0], NKV = k.extent[1], BS = k.extent[2];
    const sanic_node& tables = d->nodes[st.leaf[3]];
    std::string c;
    c += constant("T", T) + constant("NH", NH) + constant("HD", HD) + constant("NB", NB) + constant("BS", BS) + constant("REP", NH / NKV);
    c += constant("B", tables.shape[0]) + constant("M", tables.shape[1]) + constant("W", st.stream);
    c += constant("DQ", q.dtype) + constant("DC", k.dtype) + constant("DO", st.out_dtype) + "constexpr float SCALE = " + flit(d->nodes[st.leaf[6]].value) + ";\n";
    auto strides = [&](const char* n, const OperandView& o) {
        for (size_t j = 0; j < o.stride.size(); j++) c += constant((std::string(n) + std::to_string(j)).c_str(), o.stride[j]);
        c += constant((std::string(n) + "B").c_str(), o.base);
    };
    strides("Q", q), strides("K", k), strides("V", v);
    LoweredStage L;
    L.kernel_kind = "operator:paged_attn[plain]";
    L.source = std::string(kPrelude) + kElement + c + kPlain;
    Launch ln{"sanic_paged_attn", "", dim3((unsigned)((T * NH + 3) / 4)), dim3(256), 0, {}};
    for (int b : {q.buffer, k.buffer, v.buffer, tables.buffer, d->nodes[st.leaf[4]].buffer, d->nodes[st.leaf[5]].buffer, st.out_buffer})
        ln.args.push_back({Arg::BUF, b});
    L.launches.push_back(ln);
    return L;
}

}  // namespace sanic
