// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request b's rows s ≤ r < e hold its last token and its drafts; the draft behind row r is token
// x = tokens[r + 1], accepted while u[r]·q_r(x) < p_r(x). At the first refusal the token is drawn from
// max(p_r − q_r, 0), behind the last draft from p_r: the lowest t with w_0 + … + w_t > draw·Σ w. An
// accepted draft has probability min(q, p), a drawn one the rest, so together the tokens are
// distributed as the target's.
#include <algorithm>

#include "operators.h"

namespace sanic {

// One workgroup per request: the drafts' tests one per lane, then the row in runs of 8 a thread,
// summed in f64 (sums over a vocabulary lose the low bits of 24, and the drawn index with them).
static const char* kVerify = R"SRC(
typedef sanic_elem<DP>::T p_t;
typedef sanic_elem<DQ>::T q_t;
struct Args { const p_t* p; const q_t* q; const unsigned* tokens; const float *u, *draw; const unsigned* starts; unsigned *accepted, *out; };

__shared__ double part[NW];
__shared__ int found;
// exclusive prefix sum over the workgroup, in thread order
__device__ __forceinline__ double block_scan(double v, double& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double inc = v;
  for (int o = 1; o < 64; o <<= 1) {
    const double n = __shfl_up(inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 63) part[wave] = inc;
  __syncthreads();
  double before = 0.0;
  sum = 0.0;
  for (int w = 0; w < NW; w++) {
    if (w < wave) before += part[w];
    sum += part[w];
  }
  return before + inc - v;
}

extern "C" __global__ void __launch_bounds__(64 * NW) sanic_verify(Args a) {
  const int tid = threadIdx.x, lane = tid & 63;
  const long long b = blockIdx.x;
  const long long s = a.starts[b] < T ? a.starts[b] : T, e = a.starts[b + 1] < T ? a.starts[b + 1] : T;
  if (s >= e) {
    if (tid == 0) a.accepted[b] = 0;
    return;
  }
  const long long drafts = e - s - 1;
  // every wave tests the drafts, 64 at a time, up to the first that is refused
  long long n = 0;
  while (n < drafts) {
    const long long r = s + n + lane;
    bool fine = false;
    if (r + 1 < e) {
      const unsigned x = a.tokens[r + 1];
      // in f64: the product of two f32 is exact there; a NaN refuses
      if (x < V) fine = (double)a.u[r] * (QROWS ? (double)sanic_get<DQ>(a.q[QB + r * Q0 + x * Q1]) : 1.0) < (double)sanic_get<DP>(a.p[PB + r * P0 + x * P1]);
    }
    const unsigned long long no = ~__ballot(fine);
    const int run = no ? __builtin_ctzll(no) : 64;
    n += run;
    if (run < 64) break;
  }
  if (n > drafts) n = drafts;
  const long long row = s + n;
  const bool refused = n < drafts;
  const unsigned x = refused ? a.tokens[row + 1] : 0xFFFFFFFFu;
  bool rest = refused;
  auto weight = [&](long long t) -> double {
    double w = (double)sanic_get<DP>(a.p[PB + row * P0 + t * P1]);
    if (rest) {
      if (QROWS) w -= (double)sanic_get<DQ>(a.q[QB + row * Q0 + t * Q1]);
      else if (t == x) w = 0.0;
    }
    return w > 0.0 ? w : 0.0;
  };
  constexpr int TILE = 64 * NW * 8;
  double total = 0.0;
  for (int pass = 0; pass < 2; pass++) {
    double mine = 0.0;
    for (long long t0 = tid * 8; t0 < V; t0 += TILE)
      for (int i = 0; i < 8; i++)
        if (t0 + i < V) mine += weight(t0 + i);
    block_scan(mine, total);
    if (total > 0.0 || !rest) break;
    rest = false;
  }
  const double goal = (double)a.draw[b] * total;
  double before = 0.0;
  if (tid == 0) found = -1;
  int last = -1, mark = -1;
  for (long long base = 0; base < V; base += TILE) {
    const long long t0 = base + tid * 8;
    double w[8], mine = 0.0, sum;
    for (int i = 0; i < 8; i++) {
      w[i] = t0 + i < V ? weight(t0 + i) : 0.0;
      mine += w[i];
      if (w[i] > 0.0) last = (int)(t0 + i);
    }
    double run = before + block_scan(mine, sum);
    before += sum;
    if (!(before > goal)) continue;
    for (int i = 0; i < 8 && mark < 0; i++) {
      run += w[i];
      if (w[i] > 0.0 && run > goal) mark = (int)(t0 + i);
    }
    break;
  }
  // the first index over the goal; rounding (or a draw of 1) may leave none: the last with weight
  __shared__ int low, high;
  __syncthreads();
  if (tid == 0) low = 0x7FFFFFFF, high = -1;
  __syncthreads();
  if (mark >= 0) atomicMin(&low, mark);
  if (last >= 0) atomicMax(&high, last);
  __syncthreads();
  const unsigned drawn = low != 0x7FFFFFFF ? (unsigned)low : (unsigned)high;
  for (long long i = tid; i < e - s; i += 64 * NW) a.out[s + i] = i < n ? a.tokens[s + i + 1] : i == n ? drawn : 0xFFFFFFFFu;
  if (tid == 0) a.accepted[b] = (unsigned)n;
}
)SRC";

LoweredStage lower_verify_drafts(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch) {
    (void)scratch;
    OperandView p, q;
    operand_view(d, st.leaf[0], p);
    const bool has_q = st.leaf[1] >= 0;
    if (has_q) operand_view(d, st.leaf[1], q);
    else q = p;
    const int64_t T = p.extent[0], V = p.extent[1], B = d->nodes[st.leaf[4]].shape[0];
    std::string c = constant("T", T) + constant("V", V) + constant("NW", 16) + constant("QROWS", has_q) + constant("DP", p.dtype) + constant("DQ", q.dtype);
    c += constant("PB", p.base) + constant("P0", p.stride[0]) + constant("P1", p.stride[1]);
    c += constant("QB", q.base) + constant("Q0", q.stride[0]) + constant("Q1", q.stride[1]);
    LoweredStage L;
    L.kernel_kind = "operator:verify_drafts";
    L.source = std::string(kPrelude) + kElement + c + kVerify;
    Launch ln{"sanic_verify", "", dim3((unsigned)B), dim3(1024), 0, {}};
    for (int b : {p.buffer, q.buffer}) ln.args.push_back({Arg::BUF, b});
    for (int l : {2, 3, 4, 5, 6}) ln.args.push_back({Arg::BUF, d->nodes[st.leaf[l]].buffer});
    ln.args.push_back({Arg::BUF, st.out_buffer});
    L.launches.push_back(ln);
    return L;
}

}  // namespace sanic
