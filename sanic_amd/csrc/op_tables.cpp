// Block tables and slot maps of a step from the requests' lengths, and the write of the step's K and
// V rows through the slot map.
#include <algorithm>

#include "operators.h"

namespace sanic {

// One launch, no exchange between workgroups: each repeats the two prefix sums over the requests
// (lengths cut at T, then the blocks wanted) in LDS and serves its share of the rows and of the new
// blocks with a binary search in them. Bound by latency: lengths, scan, search, table entry, store.
// 8 requests 3.8 us (a launch alone is most of it), 512 requests 5.7; the lengths are a few KB, so a
// launch of its own for the sums would cost more than every workgroup's repeating them.
static const char* kTables = R"SRC(
struct Args { const unsigned *past, *fresh, *held, *free; unsigned *tables, *slots, *positions, *held_next, *starts; };

__shared__ long long wave_part[4];
// exclusive prefix sum over the workgroup's 256 threads; the total goes to `sum`
__device__ __forceinline__ long long block_scan(long long v, long long& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long inc = v;
  for (int o = 1; o < 64; o <<= 1) {
    const long long n = __shfl_up(inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 63) wave_part[wave] = inc;
  __syncthreads();
  long long before = 0;
  sum = 0;
  for (int w = 0; w < 4; w++) {
    if (w < wave) before += wave_part[w];
    sum += wave_part[w];
  }
  return before + inc - v;
}
// the last i in [0, n) with a[i] <= x, where a[0] = 0 and a does not fall: entries that share a value
// with the next one (requests without rows or blocks) are passed over
__device__ __forceinline__ int last_at_most(const unsigned* a, int n, unsigned x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// a position's slot; none where its block is, or where the slot would not fit 32 bits (it would come out
// as another, valid one)
__device__ __forceinline__ unsigned slot_in(unsigned block, unsigned long long pos) {
  const unsigned long long slot = (unsigned long long)block * BS + pos % BS;
  return block != 0xFFFFFFFFu && slot < 0xFFFFFFFFu ? (unsigned)slot : 0xFFFFFFFFu;
}

__shared__ unsigned start_of[B + 1], block_of[B + 1];

extern "C" __global__ void __launch_bounds__(256) sanic_block_tables(Args a) {
  const int tid = threadIdx.x;
  const int b0 = tid * PER < B ? tid * PER : B, b1 = b0 + PER < B ? b0 + PER : B;
  long long mine = 0, all;
  for (int b = b0; b < b1; b++) mine += a.fresh[b];
  long long at = block_scan(mine, all);
  for (int b = b0; b < b1; b++) {
    start_of[b] = (unsigned)(at < T ? at : T);
    at += a.fresh[b];
  }
  const unsigned rows = (unsigned)(all < T ? all : T);
  if (tid == 0) start_of[B] = rows;
  __syncthreads();
  // blocks wanted: what the positions up to the request's last row need beyond what it holds
  auto wanted = [&](int b) -> long long {
    const long long n = (long long)start_of[b + 1] - start_of[b], h = a.held[b];
    if (n == 0) return 0;
    long long need = ((long long)a.past[b] + n + BS - 1) / BS;
    if (need > M) need = M;
    return need > h ? need - h : 0;
  };
  const long long taken = a.held[B], left = taken < F ? F - taken : 0;
  mine = 0;
  for (int b = b0; b < b1; b++) mine += wanted(b);
  at = block_scan(mine, all);
  // the list serves the requests in their order, so the blocks got are the wanted ones' prefix
  for (int b = b0; b < b1; b++) {
    block_of[b] = (unsigned)(at < left ? at : left);
    at += wanted(b);
  }
  const unsigned grown = (unsigned)(all < left ? all : left);
  if (tid == 0) block_of[B] = grown;
  __syncthreads();
  const unsigned first = blockIdx.x * 256 + tid, step = gridDim.x * 256;
  for (unsigned b = first; b <= B; b += step) {
    a.starts[b] = start_of[b];
    a.held_next[b] = b < B ? a.held[b] + (block_of[b + 1] - block_of[b]) : (unsigned)taken + grown;
  }
  for (unsigned x = first; x < grown; x += step) {
    const int b = last_at_most(block_of, B, x);
    a.tables[(long long)b * M + a.held[b] + (x - block_of[b])] = a.free[taken + x];
  }
  for (unsigned r = first; r < rows; r += step) {
    const int b = last_at_most(start_of, B, r);
    const unsigned long long pos = (unsigned long long)a.past[b] + (r - start_of[b]);
    const unsigned long long page = pos / BS;
    const unsigned h = a.held[b];
    unsigned slot = 0xFFFFFFFFu;
    // entries beyond those held are written by this launch: they are read from the list
    if (page < h) {
      if (page < M) slot = slot_in(a.tables[(long long)b * M + page], pos);
    } else if (page - h < block_of[b + 1] - block_of[b]) {
      slot = slot_in(a.free[taken + block_of[b] + (page - h)], pos);
    }
    a.slots[r] = slot;
    a.positions[r] = (unsigned)pos;
  }
}
)SRC";

LoweredStage lower_block_tables(const sanic_program_desc* d, const sanic_stage& st) {
    auto shape = [&](int l, int j) { return d->nodes[st.leaf[l]].shape[j]; };
    const int64_t B = shape(0, 0), F = shape(3, 0), M = shape(4, 1), T = shape(5, 0);
    LoweredStage L;
    L.kernel_kind = "operator:block_tables";
    L.source = std::string(kPrelude) + constant("B", B) + constant("F", F) + constant("M", M) + constant("T", T) + constant("BS", st.stream) +
               constant("PER", (B + 255) / 256) + kTables;
    Launch ln{"sanic_block_tables", "", dim3((unsigned)std::min<int64_t>((std::max(T, B + 1) + 255) / 256, 512)), dim3(256), 0, {}};
    for (int l = 0; l < 8; l++) ln.args.push_back({Arg::BUF, d->nodes[st.leaf[l]].buffer});
    ln.args.push_back({Arg::BUF, st.out_buffer});
    L.launches.push_back(ln);
    return L;
}

// One thread per run of RUN elements of a row, K's and V's: with rows of a multiple of 8 elements and
// strides to match, 16 to 32 bytes a load and 16 a store, else one element. Bound by HBM for a
// prompt's rows (4096 rows of 8 heads of 128, bf16: 33.6 MB in 6.4 us, 5.3 TB/s, a large copy 5.2) and
// by the launch for a decode step's (8 rows: 3.5 us).
static const char* kWrite = R"SRC(
typedef sanic_elem<DS>::T src_t;
typedef sanic_elem<DD>::T dst_t;
struct Args { const src_t *k, *v; const unsigned *slots, *starts; dst_t *kc, *vc; };
struct __attribute__((packed, aligned(4))) src_run { src_t e[RUN]; };
struct __attribute__((packed, aligned(4))) dst_run { dst_t e[RUN]; };

__device__ __forceinline__ void move(const src_t* s, dst_t* p) {
  if constexpr (RUN == 1) {
    if constexpr (DS == DD) *p = *s;
    else *p = sanic_put<DD>(sanic_get<DS>(*s));
  } else {
    const src_run in = *(const src_run*)s;
    dst_run out;
    for (int i = 0; i < RUN; i++) {
      if constexpr (DS == DD) out.e[i] = in.e[i];
      else out.e[i] = sanic_put<DD>(sanic_get<DS>(in.e[i]));
    }
    *(dst_run*)p = out;
  }
}

extern "C" __global__ void __launch_bounds__(256) sanic_cache_write(Args a) {
  const long long rows = a.starts[B] < T ? a.starts[B] : T;
  for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < rows * RUNS; x += (long long)gridDim.x * 256) {
    const long long r = x / RUNS;
    const unsigned slot = a.slots[r];
    if (slot >= SLOTS) continue;
    const long long block = slot / BS, row = slot % BS;
    const int i = (int)(x % RUNS), g = i / (HD / RUN), c = i % (HD / RUN) * RUN;
    move(a.k + (KB + r * K0 + g * K1 + c * K2), a.kc + (block * CK0 + g * CK1 + row * CK2 + c * CK3));
    move(a.v + (VB + r * V0 + g * V1 + c * V2), a.vc + (block * CV0 + g * CV1 + row * CV2 + c * CV3));
  }
}
)SRC";

LoweredStage lower_cache_write(const sanic_program_desc* d, const sanic_stage& st) {
    OperandView k, v, kc, vc;
    operand_view(d, st.leaf[0], k), operand_view(d, st.leaf[1], v), operand_view(d, st.leaf[4], kc), operand_view(d, st.leaf[5], vc);
    const int64_t T = k.extent[0], NKV = k.extent[1], HD = k.extent[2], B = d->nodes[st.leaf[3]].shape[0] - 1;
    auto runs = [&](const OperandView& o) {
        bool ok = o.base % 8 == 0 && o.stride.back() == 1;
        for (size_t j = 0; j + 1 < o.stride.size(); j++) ok = ok && o.stride[j] % 8 == 0;
        return ok;
    };
    const int64_t RUN = HD % 8 == 0 && HD > 1 && runs(k) && runs(v) && runs(kc) && runs(vc) ? 8 : 1;
    LoweredStage L;
    L.kernel_kind = std::string("operator:cache_write") + (RUN == 8 ? "" : "[scalar]");
    std::string c;
    c += constant("T", T) + constant("B", B) + constant("HD", HD) + constant("BS", kc.extent[2]) + constant("SLOTS", kc.extent[0] * kc.extent[2]);
    c += constant("RUN", RUN) + constant("RUNS", NKV * HD / RUN) + constant("DS", k.dtype) + constant("DD", kc.dtype);
    auto strides = [&](const char* n, const OperandView& o) {
        for (size_t j = 0; j < o.stride.size(); j++) c += constant((std::string(n) + std::to_string(j)).c_str(), o.stride[j]);
    };
    strides("K", k), strides("V", v), strides("CK", kc), strides("CV", vc);
    c += constant("KB", k.base) + constant("VB", v.base);
    L.source = std::string(kPrelude) + kElement + c + kWrite;
    Launch ln{"sanic_cache_write", "", dim3((unsigned)std::min<int64_t>((T * (NKV * HD / RUN) + 255) / 256, 1 << 16)), dim3(256), 0, {}};
    for (int b : {k.buffer, v.buffer, d->nodes[st.leaf[2]].buffer, d->nodes[st.leaf[3]].buffer, kc.buffer, vc.buffer}) ln.args.push_back({Arg::BUF, b});
    L.launches.push_back(ln);
    return L;
}

}  // namespace sanic
