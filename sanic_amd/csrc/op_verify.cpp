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

// CHUNKS workgroups a request, each with a run of the vocabulary: every one repeats the drafts' tests
// (one a lane) to learn the row, sums its run's weights in f64 (sums over a vocabulary lose the low bits
// of 24, and with them the drawn index), and the last to arrive finds the run that the draw falls into
// from the runs' sums and reads that run again. All of a request's workgroups are on one XCD (block
// index mod 8) where the device places blocks so, and meet through its L2. Bound by HBM for a batch and
// by the chain of dependent loads (starts, tokens, tests, row, sums, run) for one request: one request
// of 128256 entries 12.4 us, 64 of them 22.5 (floor 12.7), 200 of 32003 without q 18.8; with one workgroup a
// request 213, 244 and 24.7.
static const char* kVerify = R"SRC(
typedef sanic_elem<DP>::T p_t;
typedef sanic_elem<DQ>::T q_t;
struct Args { const p_t* p; const q_t* q; const unsigned* tokens; const float *u, *draw; const unsigned* starts; unsigned *accepted, *out; double* sums; unsigned* counts; };
template <class E> struct __attribute__((packed, aligned(sizeof(E)))) Run8 { E e[8]; };

__shared__ double part[4];
__shared__ int low, high, flag;
// exclusive prefix sum over the 256 threads, in thread order
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
  for (int w = 0; w < 4; w++) {
    if (w < wave) before += part[w];
    sum += part[w];
  }
  return before + inc - v;
}

// Weights of a row: p, or what p has over q (without q rows: p but for the refused token).
struct Row {
  const p_t* p;
  const q_t* q;
  unsigned x;
  bool rest;
  __device__ __forceinline__ double of(float pv, float qv, long long t) const {
    double w = (double)pv;
    if (rest) {
      if (QROWS) w -= (double)qv;
      else if (t == x) w = 0.0;
    }
    return w > 0.0 ? w : 0.0;     // (a NaN has no weight)
  }
  __device__ __forceinline__ void load(long long t0, double (&w)[8]) const {
    if (WIDE && t0 + 8 <= V) {
      const Run8<p_t> a = *(const Run8<p_t>*)(p + t0);
      Run8<q_t> b;
      if (QROWS && rest) b = *(const Run8<q_t>*)(q + t0);
      #pragma unroll
      for (int i = 0; i < 8; i++) w[i] = of(sanic_get<DP>(a.e[i]), QROWS && rest ? sanic_get<DQ>(b.e[i]) : 0.0f, t0 + i);
    } else {
      #pragma unroll
      for (int i = 0; i < 8; i++) {
        const long long t = t0 + i;
        w[i] = t < V ? of(sanic_get<DP>(p[t * P1]), QROWS && rest ? sanic_get<DQ>(q[t * Q1]) : 0.0f, t) : 0.0;
      }
    }
  }
};
__device__ __forceinline__ long long counter_of(long long b) { return b % 8 * CSTRIDE + b / 8 * CPAD; }
constexpr long long RUN = 2048LL * TURNS;   // vocabulary entries a workgroup
__device__ __forceinline__ double run_sum(const Row& row, long long c) {
  double mine = 0.0, sum;
  #pragma unroll (TURNS < 4 ? TURNS : 4)
  for (int k = 0; k < TURNS; k++) {
    double w[8];
    row.load(c * RUN + k * 2048 + threadIdx.x * 8, w);
    #pragma unroll
    for (int i = 0; i < 8; i++) mine += w[i];
  }
  block_scan(mine, sum);
  return sum;
}

extern "C" __global__ void __launch_bounds__(256) sanic_verify(Args a) {
  const int tid = threadIdx.x, lane = tid & 63;
  // block = (group of 8 requests, run, request): a request's blocks are equal mod 8
  const long long b = (long long)blockIdx.x / (8 * CHUNKS) * 8 + blockIdx.x % 8;
  const long long c = blockIdx.x / 8 % CHUNKS;
  if (b >= B) return;
  const long long s = a.starts[b] < T ? a.starts[b] : T, e = a.starts[b + 1] < T ? a.starts[b + 1] : T;
  if (s >= e) {
    if (tid == 0 && c == 0) a.accepted[b] = 0;
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
  const bool refused = n < drafts;
  Row row{a.p + (PB + (s + n) * P0), a.q + (QB + (s + n) * Q0), refused ? a.tokens[s + n + 1] : 0xFFFFFFFFu, refused};

  double mine = run_sum(row, c);
  double* sums = a.sums + b * ((CHUNKS + 15) / 16 * 16);    // lines of its own
  if (CHUNKS > 1) {
    if (tid == 0) sums[c] = mine;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      if (ONE_XCD) {
        flag = __hip_atomic_fetch_add(a.counts + counter_of(b), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == CHUNKS - 1;
      } else {
        flag = __hip_atomic_fetch_add(a.counts + counter_of(b), 1u, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT) == CHUNKS - 1;
        if (flag) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
      }
    }
    __syncthreads();
    if (!flag) return;
    if (tid == 0) a.counts[counter_of(b)] = 0;     // the next launch's arrivals count from 0 again
  }
  // the runs' sums, PER a thread in order
  constexpr int PER = (CHUNKS + 255) / 256;
  double own[PER], total;
  auto load_sums = [&](double& at) {
    double t = 0.0;
    #pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = tid * PER + k;
      own[k] = i < CHUNKS ? (CHUNKS > 1 ? sums[i] : mine) : 0.0;
      t += own[k];
    }
    at = block_scan(t, total);
  };
  double at;
  load_sums(at);
  if (!(total > 0.0) && row.rest) {
    // p has nothing over q: the token is drawn from p (this workgroup sums it all; p and q then agree)
    row.rest = false;
    for (long long k = 0; k < CHUNKS; k++) {
      mine = run_sum(row, k);
      if (CHUNKS > 1 && tid == 0) sums[k] = mine;
    }
    __syncthreads();
    load_sums(at);
  }
  const double goal = (double)a.draw[b] * total;
  // the first run whose end is over the goal; where rounding or a draw of 1 leaves none, the last with weight
  if (tid == 0) low = 0x7FFFFFFF, high = -1;
  __syncthreads();
  int first = -1, last = -1;
  double run = at;
  #pragma unroll
  for (int k = 0; k < PER; k++) {
    run += own[k];
    if (own[k] > 0.0) {
      last = tid * PER + k;
      if (first < 0 && run > goal) first = last;
    }
  }
  if (first >= 0) atomicMin(&low, first);
  if (last >= 0) atomicMax(&high, last);
  __syncthreads();
  const int pick = low != 0x7FFFFFFF ? low : high;
  // the sum ahead of that run, from the thread that has it
  __shared__ double ahead;
  if (pick >= 0 && tid == pick / PER) {
    double x = at;
    for (int k = 0; k < pick % PER; k++) x += own[k];
    ahead = x;
  }
  __syncthreads();
  if (tid == 0) low = 0x7FFFFFFF, high = -1;
  __syncthreads();
  if (pick >= 0) {
    double before = ahead;
    int mark = -1;
    last = -1;
    for (int k = 0; k < TURNS; k++) {
      const long long t0 = pick * RUN + k * 2048 + tid * 8;
      double w[8], sum, m = 0.0;
      row.load(t0, w);
      #pragma unroll
      for (int i = 0; i < 8; i++) {
        m += w[i];
        if (w[i] > 0.0) last = (int)(t0 + i);
      }
      double x = before + block_scan(m, sum);
      before += sum;
      #pragma unroll
      for (int i = 0; i < 8; i++) {
        x += w[i];
        if (mark < 0 && w[i] > 0.0 && x > goal) mark = (int)(t0 + i);
      }
    }
    if (mark >= 0) atomicMin(&low, mark);
    if (last >= 0) atomicMax(&high, last);
  }
  __syncthreads();
  const unsigned drawn = low != 0x7FFFFFFF ? (unsigned)low : (unsigned)high;
  for (long long i = tid; i < e - s; i += 256) a.out[s + i] = i < n ? a.tokens[s + i + 1] : i == n ? drawn : 0xFFFFFFFFu;
  if (tid == 0) a.accepted[b] = (unsigned)n;
}
)SRC";

LoweredStage lower_verify_drafts(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch) {
    OperandView p, q;
    operand_view(d, st.leaf[0], p);
    const bool has_q = st.leaf[1] >= 0;
    if (has_q) operand_view(d, st.leaf[1], q);
    else q = p;
    const int64_t T = p.extent[0], V = p.extent[1], B = d->nodes[st.leaf[4]].shape[0];
    // runs of 2048 entries, or so much longer that a batch has at most 4096 workgroups (two rounds of 8 a
    // CU) and a request at most 1024. With at most 512, 1024, 2048, 4096 and 8192: 64 requests of 128256
    // entries with q 28.0, 24.3, 22.7, 23.5 and 23.4 us, 128 of them without q 36.4, 30.6, 28.4, 26.3 and
    // 28.2, 200 of 32003 in bf16 22.0, 22.9, 20.2, 19.7 and 19.3
    int64_t turns = 1;
    auto runs = [&] { return (V + 2048 * turns - 1) / (2048 * turns); };
    while (runs() > 1 && (B * runs() > 4096 || runs() > 1024)) turns *= 2;
    const int64_t chunks = runs();
    std::string c = constant("T", T) + constant("V", V) + constant("B", B) + constant("QROWS", has_q) + constant("DP", p.dtype) + constant("DQ", q.dtype);
    c += constant("PB", p.base) + constant("P0", p.stride[0]) + constant("P1", p.stride[1]) + constant("WIDE", p.stride[1] == 1 && q.stride[1] == 1);
    c += constant("QB", q.base) + constant("Q0", q.stride[0]) + constant("Q1", q.stride[1]);
    c += constant("TURNS", turns) + constant("CHUNKS", chunks) + constant("ONE_XCD", xcd_local_enabled());
    // an arrival counter a 128-byte line, or for many requests at least an XCD's on lines of their own:
    // a line that several XCDs count on goes back and forth between them (64 requests of 63 runs:
    // 46 us with the counters side by side, 26 by XCD, 23 apart)
    const int64_t cpad = B <= 256 ? 32 : 1, cstride = ((B + 7) / 8 * cpad + 31) / 32 * 32;
    c += constant("CPAD", cpad) + constant("CSTRIDE", cstride);
    LoweredStage L;
    L.kernel_kind = "operator:verify_drafts";
    L.source = std::string(kPrelude) + kElement + c + kVerify;
    Launch ln{"sanic_verify", "", dim3((unsigned)((B + 7) / 8 * 8 * chunks)), dim3(256), 0, {}};
    for (int b : {p.buffer, q.buffer}) ln.args.push_back({Arg::BUF, b});
    for (int l : {2, 3, 4, 5, 6}) ln.args.push_back({Arg::BUF, d->nodes[st.leaf[l]].buffer});
    ln.args.push_back({Arg::BUF, st.out_buffer});
    ln.args.push_back({Arg::SCRATCH, shared_scratch(scratch, B * ((chunks + 15) / 16 * 16) * 8)});
    ln.args.push_back({Arg::COUNTERS, shared_counters(8 * cstride)});
    L.launches.push_back(ln);
    return L;
}

}  // namespace sanic
