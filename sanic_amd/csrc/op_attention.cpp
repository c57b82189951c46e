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
// layout. Bound by its f32 operations and by reading every key once a row: 16 to 70 times the
// matrix-core kernel's time where both can run (a token of each of 64 requests 3848 us against 236, 4096
// rows of a prompt behind 12288 tokens 82.9 ms against 1.19).
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
  bool falls = false;
  for (int i = lane; i < B; i += 64) falls |= a.starts[i + 1] < T && a.starts[i + 1] < a.starts[i];
  if (__any(falls)) return;
  int b = 0, hi_b = B;   // the last request that starts at or before r
  while (hi_b - b > 1) {
    const int mid = (b + hi_b) >> 1;
    if (a.starts[mid] <= r) b = mid; else hi_b = mid;
  }
  if (r < a.starts[b] || r >= a.starts[b + 1]) return;
  const long long p = (long long)a.past[b] + (r - a.starts[b]);
  const long long most = (long long)M * BS, end = p + 1 < most ? p + 1 : most;
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
    for (int i = 0; i < DV; i++) o[i] = __builtin_fabsf(o[i]) == __builtin_huge_valf() ? o[i] : o[i] * c;   // (a factor of 0 leaves it infinite)
    w_of[wave][lane] = w;
    page_of[wave][lane] = page;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int x = 0; x < 64; x++) {
      const unsigned pg = page_of[wave][x];
      if (pg >= NB) continue;   // a masked place's value may be anything, NaN among it
      const kv_t* v = a.v + (VB + pg * V0 + g * V1 + (base + x) % BS * V2);
      const float wx = w_of[wave][x];
      for (int i = 0; i < DV; i++)
        if (lane + 64 * i < HD) {
          // (a value that is not finite stays what it is, also at a weight that is 0 in 32 bits)
          const float y = sanic_get<DC>(v[(lane + 64 * i) * V3]);
          o[i] = __builtin_fabsf(y) < __builtin_huge_valf() ? __builtin_fmaf(wx, y, o[i]) : o[i] + y;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  for (int i = 0; i < DV; i++)
    if (lane + 64 * i < HD) a.o[(r * NH + h) * HD + lane + 64 * i] = sanic_put<DO>(sum == 0.0f ? 0.0f : o[i] / sum);
}
)SRC";

// The matrix-core kernel: bf16 or f16 queries and caches, heads of a multiple of 16 up to 256.
//
// A workgroup (4 waves) takes one key head's rows of one request: the NH / NKV query heads that read
// it and the request's new rows are one axis (packed row = row · REP + head), since they share every
// key. Few rows (up to DR = 32, a decoded token or its drafts): the four waves split a tile's keys in
// groups of 16 (and, with tiles of 32 keys, the value dims) and meet in LDS at the end. More rows: a
// workgroup takes PR = 128 of them, 32 a wave, and each wave goes over all keys. Either way tiles of
// TK keys come straight from the pages into a ring of LDS buffers (16 bytes a lane, no register
// staging), addressed through the item's part of the block table in LDS.
//
// Work is split over keys too. Request lengths are known on the device alone, so every workgroup sums
// the requests' key tiles and derives the same plan. The few-row requests' tiles, one request behind
// the other, are cut into as many equal runs as workgroups are resident: a run may end one request and
// begin the next, and no workgroup has more than another (24 requests of 5 drafts: 55 us, now 50; an item a
// workgroup, with the longest request's items last, 68). Many-row tiles are split into parts over the
// keys. Either way the partials fit the scratch. The parts of one row meet in the workgroup that
// arrives last, which adds them in split order. The arrivals are relaxed where a key head's workgroups
// share an XCD, whose L2 they meet in (a release writes that L2 back: 103 us instead of 68).
//
// Bound by HBM for decoded tokens: 64 requests of 32/8 heads of 128, 1.2 GB of cache, 236 us, 5.1 TB/s
// (a large copy: 5.2); 10.8 us for one request, a chain of dependent loads. Bound by matrix and vector
// instructions for a prompt (38% and 36% of the SIMDs' cycles): 4096 rows of 32/8 heads of 128 behind 12288
// tokens, 1107 to 1187 us by the card, 811 to 869 TFLOP/s (a large product: 1235). What brought
// it there from 2911 us: tiles as blocks of 1 KB whose reads differ by constant offsets, and eight
// transposed reads to one wait (1795); page addresses in scalar registers (1157; the 64 requests 310 to
// 236). Finding sums that are not finite, and what a second pass over such rows needs, took 0.5 us of a
// single request's call and 2% of that prompt's.
//
// Scores are computed transposed (Sᵀ = K·Qᵀ), so a lane owns one row's column: softmax statistics are
// lane-local plus two lane swaps, and Sᵀ's layout is the B operand of Oᵀ = Vᵀ·P as it stands. Softmax
// runs in base 2, t = s·(scale·log2 e); the reference moves only when a tile's maximum exceeds it by
// 8, so weights reach 2^8 and rescaling is rare; sums come from the matrix cores (ones times P), of the
// weights as rounded for the product.
static const char* kMfma = R"SRC(
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef sanic_elem<DO>::T o_t;
struct Args { const unsigned short *q, *k, *v; const unsigned *tables, *starts, *past; o_t* o; float* part; unsigned* counts; };

constexpr bool HALF = DQ == 2;
constexpr int CH = HD / 8, CG = (CH + 3) / 4;    // 16-byte chunks of a key's row, and 64-byte groups of them
constexpr int DSTEP = CG, DT = HD / 16;          // products over 32 head dims; value tiles of 16 dims
// tiles of TK keys in a ring of ST
template <int TK_, int ST_> struct Ring {
  static constexpr int TK = TK_, ST = ST_;
  static constexpr int LOADS = (TK / 16 * CG + 3) / 4;   // 16-byte loads a lane for a tile's keys, and its values
  static constexpr int TILE = LOADS * 4 * 512;           // elements of a staged tile, surplus loads included
  static constexpr int SIZE = ST * 2 * TILE;
  static __device__ __forceinline__ int at(int buf, int value) { return (buf * 2 + value) * TILE; }
};
typedef Ring<FEW_TK, FEW_ST> Few;
typedef Ring<MANY_TK, MANY_ST> Many;
constexpr int KG = FEW_TK / 16, DH = 4 / KG, DTH = DH == 1 ? DT : (DT + 3) / 4 * 2;   // few rows: key groups, dim parts
static_assert(KG * 32 * HD * 4 <= Few::SIZE * 2 && 256 * 24 <= Few::SIZE * 2);
constexpr int RING = Few::SIZE > Many::SIZE || !PITEMS ? Few::SIZE : Many::SIZE;
constexpr int MBS = M * BS;                      // positions a block table can hold
constexpr float NEG_INF = -__builtin_huge_valf();

__device__ __forceinline__ f32x4 mma32(s16x8 x, s16x8 y, f32x4 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, x), __builtin_bit_cast(b16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(s16x4 x, s16x4 y, f32x4 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, x), __builtin_bit_cast(f16x4, y), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x, y, c, 0, 0, 0);
}
// four values rounded to the matrix cores' type (ties to even), and what the rounding left
__device__ __forceinline__ u32x2 pack(f32x4& x) {
  u32x2 out;
  #pragma unroll
  for (int e = 0; e < 2; e++) {
    if constexpr (HALF) {
      const f16x2 h = {(_Float16)x[2 * e], (_Float16)x[2 * e + 1]};
      x[2 * e] -= (float)h[0], x[2 * e + 1] -= (float)h[1];
      out[e] = __builtin_bit_cast(unsigned, h);
    } else {
      const unsigned h = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x[2 * e], x[2 * e + 1]}, b16x2));
      x[2 * e] -= __uint_as_float(h << 16), x[2 * e + 1] -= __uint_as_float(h & 0xFFFF0000u);
      out[e] = h;
    }
  }
  return out;
}
__device__ __forceinline__ float quad_max(float v) {  // over the 4 lanes of a row's column
  return sanic_rows_max(v);
}
// A staged tile is made of blocks of 16 rows × 4 chunks (1 KB, one load a lane: 64 contiguous bytes of
// each row), [row group][chunk group]; inside a block the chunks of a row are swapped by the row, so
// that rows a wave reads at one dim lie in different banks, and a lane's place in a block is the same
// in all of them: reads differ by constant offsets.
__device__ __forceinline__ int in_block(int row, int c) { return ((row & 15) * 4 + ((c & 3) ^ (row >> 1 & 3))) * 8; }
__device__ __forceinline__ int spot(int row, int c) { return ((row >> 4) * CG + (c >> 2)) * 512 + in_block(row, c); }
__device__ __forceinline__ int clamp_pos(long long p) { return p < 0 ? 0 : p > MBS ? MBS : (int)p; }

// (one object: with several, the compiler waits for every load into LDS before any read of it)
__shared__ struct {
  __attribute__((aligned(1024))) unsigned short ring[RING];
  unsigned pages[PAGES];
  unsigned long long odd_keys;
  int holes, last_arrival, not_finite;
} lds;

// ── what this workgroup does ──────────────────────────────────────────────────────────────────────
struct Item {
  int b, tile, split, splits, rows, slot, count;
  long long start, past;
};
struct Req {
  long long start, past;
  int rows, tiles, kt;   // packed rows; workgroups of PR of them (0: few rows, D below); key tiles
  bool falls;            // the request ends before it starts
};
__device__ __forceinline__ Req request(const Args& a, int b) {
  Req q{0, 0, 0, 0, 0, false};
  if (b >= B) return q;
  const long long s = a.starts[b] < T ? a.starts[b] : T, e = a.starts[b + 1] < T ? a.starts[b + 1] : T;
  q.falls = e < s;
  if (e <= s) return q;
  q.start = s, q.past = a.past[b];
  q.rows = (int)(e - s) * REP;
  q.tiles = q.rows <= DR ? 0 : (q.rows + PR - 1) / PR;
  const int hi = clamp_pos(q.past + (e - s)), lo = W ? clamp_pos(q.past + 1 - W) : 0;
  const int tk = q.tiles ? MANY_TK : FEW_TK, kt = (hi + tk - 1) / tk - lo / tk;
  q.kt = kt > 1 ? kt : 1;
  return q;
}
__device__ __forceinline__ int pick(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ long long pick(long long v, int lane) {
  return (long long)((unsigned long long)(unsigned)pick((int)(v >> 32), lane) << 32 | (unsigned)pick((int)v, lane));
}
__device__ __forceinline__ int scan64(int v) {  // inclusive, over the wave
  for (int o = 1; o < 64; o <<= 1) {
    const int n = __shfl_up(v, o);
    if ((threadIdx.x & 63) >= o) v += n;
  }
  return v;
}
__device__ __forceinline__ int many_splits(int kt, int part) {
  const int s = (kt + part - 1) / part;
  return s < MOST ? s : MOST;
}
// What every wave of every workgroup computes alike from the lengths. Few-row requests' key tiles, one
// request behind the other, are cut into equal runs of `run` tiles, one a workgroup; many-row tiles are
// split into parts of `part` key tiles each.
struct Plan {
  int run, part, items, stride;    // items: of the many-row requests; stride: rows of a few-row partial
  bool none;                       // starts fall: requests overlap, and may be more than the grid has room for
};
__device__ __forceinline__ Plan make_plan(const Args& a, Req& q) {
  const int lane = threadIdx.x & 63;
  float ud = 0, umax = 0, rmax = 0, up = 0, tp = 0;
  bool falls = false;
  for (int b0 = 0; b0 < B; b0 += 64) {
    q = request(a, b0 + lane);
    falls |= q.falls;
    if (q.tiles == 0) {
      ud += q.kt;
      umax = __builtin_fmaxf(umax, q.kt), rmax = __builtin_fmaxf(rmax, q.rows);
    } else {
      up += (float)q.tiles * q.kt, tp += q.tiles;
    }
  }
  ud = sanic_wave_sum(ud), umax = sanic_wave_max(umax), rmax = sanic_wave_max(rmax);
  Plan p;
  p.none = __any(falls);
  // whole 128-byte lines of statistics and sums: the workgroup that adds one request's parts reads no line
  // that holds another's, which its CU's L1 would keep as it was and a later join there would read
  p.stride = (__builtin_amdgcn_readfirstlane((int)rmax) + LINE - 1) / LINE * LINE;
  // as many workgroups as run at once, or as their partials (two of `stride` rows each) have room, or as
  // one request's parts may be for the workgroup that adds them (about MOST)
  float groups = FEW_GROUPS;
  if (p.stride > 0) groups = __builtin_fminf(groups, __builtin_floorf((float)DROWS / (2.0f * (float)p.stride)));
  const float run = __builtin_fmaxf(ud / groups, umax / (float)MOST);
  // (the sums are f32: 1.001 covers their roundings)
  p.run = __builtin_amdgcn_readfirstlane((int)__builtin_fmaxf(1.0f, __builtin_ceilf(run * 1.001f)));
  p.part = 1 << 30, p.items = 0;
  if (PITEMS) {
    up = sanic_wave_sum(up), tp = sanic_wave_sum(tp);
    if (2.0f * tp <= (float)PSPLIT)
      // (no room beside one tile: as good as never)
      p.part = __builtin_amdgcn_readfirstlane((int)__builtin_fminf(1e9f, __builtin_fmaxf(1.0f, __builtin_ceilf(up / ((float)PSPLIT - tp - 1.0f) * 1.001f))));
    for (int b0 = 0; b0 < B; b0 += 64) {
      if (B > 64) q = request(a, b0 + lane);
      p.items += pick(scan64(q.tiles * many_splits(q.kt, p.part)), 63);
    }
  }
  return p;
}
// The many-row item `it`.
__device__ __forceinline__ void find_many(const Args& a, const Plan& p, Req& q, int it, Item& o) {
  const int lane = threadIdx.x & 63;
  int before = 0, tiles_before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    if (B > 64) q = request(a, b0 + lane);
    const int splits = many_splits(q.kt, p.part), mine = q.tiles * splits, inc = before + scan64(mine), tinc = scan64(q.tiles);
    const unsigned long long who = __ballot(mine > 0 && it >= inc - mine && it < inc);
    if (who) {
      const int l = __builtin_ctzll(who), x = it - pick(inc - mine, l), tiles = pick(q.tiles, l);
      o.b = b0 + l, o.splits = pick(splits, l), o.rows = pick(q.rows, l);
      o.tile = tiles - 1 - x / o.splits;     // the last rows see most
      o.split = x % o.splits;
      o.slot = DROWS + (it - o.split) * PR;
      o.count = B + tiles_before + pick(tinc, l) - tiles + o.tile;
      o.start = pick(q.start, l), o.past = pick(q.past, l);
      return;
    }
    before = pick(inc, 63), tiles_before += pick(tinc, 63);
  }
}

// ── tiles of keys and values ──────────────────────────────────────────────────────────────────────
struct Stream {
  const Args& a;
  const unsigned* table;
  int tid, g, first_page, last_page, base;   // the thread; the pages seen by any row; the first page in LDS
  const unsigned short *k, *v;

  // the block table from page p on into LDS (every thread, between two barriers)
  __device__ __forceinline__ void pages_from(int p) {
    base = p;
    bool hole = false;
    for (int i = threadIdx.x; i < PAGES; i += 256) {
      const int at = p + i;
      unsigned x = at <= last_page ? table[at] : 0xFFFFFFFFu;
      hole |= x >= NB && at >= first_page && at <= last_page;
      lds.pages[i] = x;
    }
    if (hole) lds.holes = 1;
  }
  template <class R> __device__ __forceinline__ bool covers(int t0) const { return t0 / BS >= base && (t0 + R::TK - 1) / BS < base + PAGES; }
  template <class R> __device__ __forceinline__ void fetch(int t0, int buf) const {
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = lane >> 2, c = (lane & 3) ^ (row >> 1 & 3);
    // 16 rows of one page: its address is the wave's, a lane's part of it the same in every tile
    unsigned page_of[R::LOADS];
    #pragma unroll
    for (int u = 0; u < R::LOADS; u++) {
      unsigned group = (unsigned)(u * 4 + wave) / CG;
      if (R::TK / 16 * CG % 4 && group >= R::TK / 16) group = R::TK / 16 - 1;
      if (BS % 16 == 0) page_of[u] = lds.pages[((unsigned)t0 + group * 16) / BS - base];
    }
    #pragma unroll
    for (int u = 0; u < R::LOADS; u++) {
      const unsigned n = u * 4 + wave;
      unsigned group = n / CG;
      const int cg = n % CG * 4;
      int chunk = c;
      if (R::TK / 16 * CG % 4 && group >= R::TK / 16) group = R::TK / 16 - 1;
      if (CH % 4 && cg + c >= CH) chunk = CH - 1 - cg;    // (read as 0 by key_run)
      const unsigned key = (unsigned)t0 + group * 16;
      // a page that is none is read as block 0 and masked
      const char *kp, *vp;
      if (BS % 16 == 0) {
        const unsigned page = __builtin_amdgcn_readfirstlane(page_of[u]);
        const long long pg = page < NB ? page : 0, in = key % BS;
        kp = (const char*)(k + (pg * K0 + in * K2 + cg * 8)) + (unsigned)(row * K2 + chunk * 8) * 2;
        vp = (const char*)(v + (pg * V0 + in * V2 + cg * 8)) + (unsigned)(row * V2 + chunk * 8) * 2;
      } else {
        const unsigned page = lds.pages[(key + row) / BS - base];
        const long long pg = page < NB ? page : 0, in = (key + row) % BS;
        kp = (const char*)(k + (pg * K0 + in * K2 + (cg + chunk) * 8));
        vp = (const char*)(v + (pg * V0 + in * V2 + (cg + chunk) * 8));
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)kp, (__attribute__((address_space(3))) void*)&lds.ring[R::at(buf, 0) + n * 512], 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vp, (__attribute__((address_space(3))) void*)&lds.ring[R::at(buf, 1) + n * 512], 16, 0, 0);
    }
  }
  // the keys of a tile that are in no block of the pool, a bit each
  template <int TK> __device__ __forceinline__ unsigned long long missing(int t0) const {
    unsigned long long out = 0;
    for (int p = t0 / BS; p <= (t0 + TK - 1) / BS; p++) {
      if (p < first_page || p > last_page || table[p] < NB) continue;
      const int from = p * BS - t0, to = from + BS;
      for (int r = from > 0 ? from : 0; r < (to < TK ? to : TK); r++) out |= 1ull << r;
    }
    return out;
  }
};

template <class R>
__device__ __forceinline__ void need(Stream& st, int t0) {
  if (st.covers<R>(t0)) return;
  __syncthreads();
  st.pages_from(t0 / BS);
  __syncthreads();
}
// The first tiles under way. The query rows are waited for before them (behind the block table, which
// is anyway): the compiler would otherwise wait for them, and so for every tile, inside the loop.
template <class R, int RT>
__device__ __forceinline__ void begin(Stream& st, int t_first, int t_last, s16x8 (&q)[RT][DSTEP]) {
  if (threadIdx.x == 0) lds.holes = 0, lds.not_finite = 0;
  __syncthreads();
  if (t_first < t_last) st.pages_from(t_first * R::TK / BS);
  #pragma unroll
  for (int t = 0; t < RT; t++)
    #pragma unroll
    for (int d = 0; d < DSTEP; d++) asm volatile("" : "+v"(q[t][d]));
  __syncthreads();
  #pragma unroll
  for (int i = 0; i < R::ST - 1; i++) {
    if (t_first + i >= t_last) break;
    need<R>(st, (t_first + i) * R::TK);
    st.fetch<R>((t_first + i) * R::TK, i);
  }
}
// Tile t has arrived in every wave's part of it, and the tile before it is done with: the next tile
// under way takes its place.
template <class R>
__device__ __forceinline__ void turn(Stream& st, int t, int t_last, int buf) {
  const int left = t_last - 1 - t;      // tiles behind it that are under way: up to ST − 2
  if (R::ST > 3 && left >= 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * 2 * R::LOADS) : "memory");
  else if (R::ST > 2 && left >= 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * R::LOADS) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if (t + R::ST - 1 < t_last) {
    need<R>(st, (t + R::ST - 1) * R::TK);
    st.fetch<R>((t + R::ST - 1) * R::TK, buf == 0 ? R::ST - 1 : buf - 1);
  }
}

__device__ __forceinline__ s16x8 key_run(int tile, int group, int step, int l16, int lq) {
  s16x8 x = *(const s16x8*)&lds.ring[tile + (group * CG + step) * 512 + in_block(l16, lq)];
  // behind a head's end stand copies of other dims, which need not be finite, and the query's 0 would not
  // take those out of the product
  if (HD % 32 && step == DSTEP - 1 && step * 4 + lq >= CH) x = (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
  return x;
}
// Transposed reads of 16 keys × 16 value dims: a lane gets 4 keys of one dim. A lane's place in a block
// for an even tile of dims; for an odd one it is 32 bytes further or back (two chunks, swapped alike).
__device__ __forceinline__ unsigned value_at(int tile, int l16, int lq) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned short*)&lds.ring[tile + in_block(lq * 4 + (l16 >> 2), l16 >> 1 & 1) + (l16 & 1) * 4];
}
// (waited for in the same statement: the compiler takes an asm output as written at once)
template <int I0, int I1>
__device__ __forceinline__ void tr_read4(unsigned even, s16x4& r0, s16x4& r1, s16x4& r2, s16x4& r3) {
  asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %5 offset:%6\n\t"
               "ds_read_b64_tr_b16 %2, %4 offset:%7\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3) : "v"(even), "v"(even ^ 32u), "n"(I0), "n"(I1) : "memory");
}
template <int I0, int I1, int I2, int I3>
__device__ __forceinline__ void tr_read8(unsigned even, s16x4 (&r)[8]) {
  asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %9 offset:%10\n\t"
               "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %9 offset:%11\n\t"
               "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
               "ds_read_b64_tr_b16 %6, %8 offset:%13\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
               : "v"(even), "v"(even ^ 32u), "n"(I0), "n"(I1), "n"(I2), "n"(I3) : "memory");
}
__device__ __forceinline__ bool odd_value(unsigned short x) { return HALF ? (x & 0x7C00) == 0x7C00 : (x & 0x7F80) == 0x7F80; }

// Sums scaled to another reference: an infinite one stays infinite where the factor is 0 in 32 bits.
__device__ __forceinline__ f32x4 scaled(f32x4 v, float f) {
  #pragma unroll
  for (int r = 0; r < 4; r++) v[r] = __builtin_fabsf(v[r]) == __builtin_huge_valf() ? v[r] : v[r] * f;
  return v;
}

// One column of scores into weights: s holds the products of the tile's keys row0 + 16·kt + r, of which
// the row sees those in [lo, hi) that are no holes, and leaves as 2^(t − m). `factor` is what the row's earlier sums are scaled by.
// A tile's maximum may exceed the reference by `lead`.
template <int N>
__device__ __forceinline__ void weigh(f32x4 (&s)[N], bool full, unsigned long long holes, int row0, int lo, int hi, float lead, float& m, float& factor) {
  float top = NEG_INF;
  if (full) {
    #pragma unroll
    for (int kt = 0; kt < N; kt++) top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(top, s[kt][0]), __builtin_fmaxf(s[kt][1], s[kt][2])), s[kt][3]);
    top *= C2;
  } else {
    #pragma unroll
    for (int kt = 0; kt < N; kt++)
      #pragma unroll
      for (int r = 0; r < 4; r++) {
        const int key = row0 + kt * 16 + r;
        const bool seen = key >= lo && key < hi && !(holes >> key & 1);
        s[kt][r] = seen ? s[kt][r] * C2 : NEG_INF;
        top = __builtin_fmaxf(top, s[kt][r]);
      }
  }
  factor = 1.0f;
  if (!__all(top <= m + lead && m > NEG_INF)) {
    top = quad_max(top);
    const float to = top > m + lead ? top : m;
    // (without a reference so far there are no sums but 0 and what is not finite)
    factor = to == m || m == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    m = to;
  }
  // nothing seen so far, or scores of −inf alone: their weights are 0, 2^(−inf − 0)
  const float ref = m == NEG_INF ? 0.0f : m;
  // (a branch for the whole tile, or a choice for each score, by what the compiler makes of them: heads of
  // 128, 4096 rows 1187 us against 1238; heads of 64, a mixed batch 65.8 against 55.2)
  if (HD > 64 && full) {
    #pragma unroll
    for (int kt = 0; kt < N; kt++)
      #pragma unroll
      for (int r = 0; r < 4; r++) s[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], C2, -ref));
  } else {
    #pragma unroll
    for (int kt = 0; kt < N; kt++)
      #pragma unroll
      for (int r = 0; r < 4; r++) s[kt][r] = __builtin_amdgcn_exp2f(full ? __builtin_fmaf(s[kt][r], C2, -ref) : s[kt][r] - ref);
  }
}

// Values that nobody in the workgroup sees become 0 (0·NaN would reach every row of the product);
// where one that is seen is not finite, its key's bit is returned, and it is 0 in the tile: add_odd
// adds it to the rows that see it. Tiles that every row sees whole are not cleaned: there a value that
// is not finite goes through the product, which may make NaN of an infinite one (by a weight that is 0
// in 32 bits, by the negative rest of a weight's first term). Rows whose sums come out not finite are
// computed again with every tile cleaned, and with the largest score so far as the reference (a lead of
// 2^8 could take sums of values near the end of the range past it). Rows [row0, row0 + rows) × chunks [c0, c0 + chunks), of which any row
// sees [lo, hi) (rows counted from the tile's first key).
__device__ __forceinline__ unsigned long long clean(int tile, unsigned long long holes, int row0, int rows, int c0, int chunks, int lo, int hi, int part, int parts) {
  unsigned long long odd = 0;
  for (int i = part; i < rows * chunks; i += parts) {
    const int row = row0 + i / chunks;
    s16x8* p = (s16x8*)&lds.ring[tile + spot(row, c0 + i % chunks)];
    s16x8 x = *p;
    const bool dead = row < lo || row >= hi || (holes >> row & 1);
    bool change = dead;
    #pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool o = odd_value((unsigned short)x[e]);
      change |= o;
      if (o && !dead) odd |= 1ull << row;
      if (o || dead) x[e] = 0;
    }
    if (change) *p = x;
  }
  return odd;
}
// The values of the tile's keys `odd` that are not finite, to the rows that see those keys: a weight above
// 0, however small, leaves such a value what it is.
template <int D>
__device__ __forceinline__ void add_odd(const Stream& st, unsigned long long odd, int t0, int lo, int hi, f32x4 (&o)[D], int dt0, int lq) {
  while (odd) {
    const int row = __builtin_ctzll(odd), key = t0 + row;
    odd &= odd - 1;
    const bool seen = row >= lo && row < hi;
    const unsigned page = st.table[key / BS];
    const unsigned short* v = st.v + ((long long)page * V0 + key % BS * V2);
    #pragma unroll
    for (int d = 0; d < D; d++) {
      const int col = (dt0 + d) * 16 + lq * 4;
      if (col >= HD) continue;
      struct __attribute__((packed, aligned(4))) run { unsigned short e[4]; };
      const run y = *(const run*)(v + col);
      #pragma unroll
      for (int r = 0; r < 4; r++)
        o[d][r] += seen && odd_value(y.e[r]) ? sanic_get<DQ>(__builtin_bit_cast(sanic_elem<DQ>::T, y.e[r])) : 0.0f;
    }
  }
}
template <int N> __device__ __forceinline__ bool not_finite(const f32x4 (&o)[N], const f32x4& sum) {
  f32x4 x = sum * 0.0f;
  #pragma unroll
  for (int d = 0; d < N; d++)
    #pragma unroll
    for (int r = 0; r < 4; r++) x[r] = __builtin_fmaf(o[d][r], 0.0f, x[r]);
  return (x[0] + x[1]) + (x[2] + x[3]) != 0.0f;     // NaN
}

// ── the parts of a row ────────────────────────────────────────────────────────────────────────────
// part: DROWS + PSPLIT·PR rows a key head, of HD sums and, behind all of those, the maximum and the sum
__device__ __forceinline__ float* part_sums(const Args& a, int g, int slot) { return a.part + ((long long)g * SLOTS + slot) * HD; }
__device__ __forceinline__ float* part_stats(const Args& a, int g, int slot) { return a.part + (long long)NKV * SLOTS * HD + ((long long)g * SLOTS + slot) * 2; }
__device__ __forceinline__ long long out_at(const Item& it, int g, int row) {
  return ((it.start + row / REP) * NH + g * REP + row % REP) * (long long)HD;
}
__device__ __forceinline__ void put4(o_t* p, f32x4 v) {
  if constexpr (DO == 1) {
    struct __attribute__((packed, aligned(4))) run { f32x4 v; };
    ((run*)p)->v = v;
  } else {
    struct __attribute__((packed, aligned(4))) run { o_t e[4]; };
    run x;
    for (int e = 0; e < 4; e++) x.e[e] = sanic_put<DO>(v[e]);
    *(run*)p = x;
  }
}
// The splits of rows [row0, row0 + rows) meet: the last workgroup to arrive adds them in their order.
// Split s of row r stands at slot + s·stride + r, of the first split (few rows) one place before.
__device__ __forceinline__ void meet(const Args& a, const Item& it, int g, int row0, int rows, int stride, int first) {
  const int tid = threadIdx.x, splits = it.splits;
  auto place = [&](int s) { return it.slot + (s == 0 ? first : s * stride); };
  unsigned* cnt = a.counts + ((long long)g * COUNTS + it.count * CPAD);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    if (ONE_XCD) {
      lds.last_arrival = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)splits - 1u;
    } else {
      lds.last_arrival = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)splits - 1u;
      if (lds.last_arrival) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    }
  }
  __syncthreads();
  if (!lds.last_arrival) return;
  if (tid == 0) *cnt = 0;      // the next launch's arrivals count from 0 again
  // a thread's sums: 4 value dims of a row over the splits, statistics and sums loaded together; with few
  // of them, teams take every teams-th split each and meet in LDS
  const int units = rows * (HD / 4), teams = units >= 256 ? 1 : 256 / units;
  const int team = teams == 1 ? 0 : tid / units;
  for (int u = teams == 1 ? tid : tid % units; u < units; u += 256) {
    const int r = u / (HD / 4), d = u % (HD / 4) * 4;
    f32x4 acc = {0, 0, 0, 0};
    float m = NEG_INF, l = 0.0f;
    auto add = [&](float m2, float l2, f32x4 v, bool careful) {
      const float to = __builtin_fmaxf(m, m2), ref = to == NEG_INF ? 0.0f : to;   // (a split that saw nothing has weight 0)
      const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
      acc = careful ? scaled(acc, f) + scaled(v, f2) : acc * f + v * f2;
      l = l * f + l2 * f2;
      m = to;
    };
    auto add_part = [&](int s, bool careful) {
      const f32x2 x = *(const f32x2*)part_stats(a, g, place(s) + r);
      add(x[0], x[1], *(const f32x4*)(part_sums(a, g, place(s) + r) + d), careful);
    };
    // where the sums are NaN, an infinite one may have met a factor of 0: they are added once more, with care
    // (with care at once a single request's call takes 0.5 us of 11 more)
    auto nan = [&] { const float x = (acc[0] + acc[1]) + (acc[2] + acc[3]); return x != x; };
    if (team < teams) {
      #pragma unroll 4
      for (int s = team; s < splits; s += teams) add_part(s, false);
      if (nan()) {
        acc = (f32x4){0, 0, 0, 0}, m = NEG_INF, l = 0.0f;
        #pragma unroll 1
        for (int s = team; s < splits; s += teams) add_part(s, true);
      }
    }
    if (teams > 1) {
      f32x4* sums = (f32x4*)lds.ring;
      f32x2* stats = (f32x2*)(sums + 256);
      sums[tid] = acc;
      stats[tid] = (f32x2){m, l};
      __syncthreads();
      if (team != 0) break;
      auto add_team = [&](int k, bool careful) { add(stats[k * units + tid][0], stats[k * units + tid][1], sums[k * units + tid], careful); };
      for (int k = 1; k < teams; k++) add_team(k, false);
      if (nan()) {
        acc = (f32x4){0, 0, 0, 0}, m = NEG_INF, l = 0.0f;
        #pragma unroll 1
        for (int k = 0; k < teams; k++) add_team(k, true);
      }
    }
    put4(a.o + out_at(it, g, row0 + r) + d, l == 0.0f ? (f32x4){0, 0, 0, 0} : acc / l);
  }
}

// a lane's part of a query row; a negative scale is the query's
__device__ __forceinline__ void read_row(const unsigned short* q, int lq, s16x8 (&x)[DSTEP]) {
  struct __attribute__((packed, aligned(4))) run { s16x8 v; };
  #pragma unroll
  for (int s = 0; s < DSTEP; s++) {
    x[s] = (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
    if (HD % 32 == 0 || s * 4 + lq < CH) x[s] = ((const run*)(q + (s * 4 + lq) * 8))->v;
    if (FLIP) x[s] ^= (short)0x8000;
  }
}

// the values of 16 keys, four tiles of dims at a time (a last tile's read may be of the tile before it)
template <int D>
__device__ __forceinline__ void few_values(unsigned at, s16x4 (&vt)[(DTH + 3) / 4 * 4]) {
  tr_read4<D / 2 * 1024, (D / 2 + 1 < CG ? D / 2 + 1 : D / 2) * 1024>(at, vt[D], vt[D + 1], vt[D + 2], vt[D + 3]);
  if constexpr (D + 4 < DTH) few_values<D + 4>(at, vt);
}

// ── few rows: the waves split the tile's keys ─────────────────────────────────────────────────────
template <int RT>
__device__ __forceinline__ bool few_rows(const Args& a, const Item& it, int stride, int g, Stream& st, int t_first, int t_last, int lo_all, int hi_all, int full_lo, int full_hi, bool careful) {
  constexpr int TK = FEW_TK;
  const int tid = st.tid, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lq = lane >> 4;
  const int kg = wave % KG, dh = wave / KG, dt0 = dh * DTH;
  s16x8 qf[RT][DSTEP];
  int lo[RT], hi[RT];
  #pragma unroll
  for (int t = 0; t < RT; t++) {
    int row = t * 16 + l16;
    if (row >= it.rows) row = it.rows - 1;
    const unsigned short* q = a.q + (QB + (it.start + row / REP) * Q0 + (g * REP + row % REP) * Q1);
    read_row(q, lq, qf[t]);
    hi[t] = clamp_pos(it.past + row / REP + 1);
    lo[t] = W ? clamp_pos(it.past + row / REP + 1 - W) : 0;
  }
  f32x4 o[RT][DTH], sum[RT];
  float m[RT];
  #pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = NEG_INF, sum[t] = (f32x4){0, 0, 0, 0};
    #pragma unroll
    for (int d = 0; d < DTH; d++) o[t][d] = (f32x4){0, 0, 0, 0};
  }
  begin<Few>(st, t_first, t_last, qf);
  const short one = HALF ? (short)0x3C00 : (short)0x3F80;
  const s16x4 ones = {one, one, one, one};
  int buf = 0;
  for (int i = t_first; i < t_last; i++) {
    const int t0 = i * TK;
    turn<Few>(st, i, t_last, buf);
    const unsigned long long holes = lds.holes ? st.missing<TK>(t0) : 0;
    const bool full = !careful && t0 >= full_lo && t0 + TK <= full_hi && !holes;
    unsigned long long odd = 0;
    if (!full) {
      const int c0 = dt0 * 2, c1 = (dt0 + DTH) * 2 < CH ? (dt0 + DTH) * 2 : CH;
      odd = clean(Few::at(buf, 1), holes, kg * 16, 16, c0, c1 - c0, lo_all - t0, hi_all - t0, lane, 64);
      for (int x = 1; x < 64; x <<= 1) odd |= __shfl_xor(odd, x);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    s16x4 vt[(DTH + 3) / 4 * 4];
    #pragma unroll
    for (int t = 0; t < RT; t++) {
      f32x4 s[1] = {{0, 0, 0, 0}};
      #pragma unroll
      for (int d = 0; d < DSTEP; d++) s[0] = mma32(key_run(Few::at(buf, 0), kg, d, l16, lq), qf[t][d], s[0]);
      float factor;
      weigh<1>(s, full, holes, kg * 16 + lq * 4, lo[t] - t0, hi[t] - t0, careful ? 0.0f : 8.0f, m[t], factor);
      if (!__all(factor == 1.0f)) {
        sum[t] *= factor;
        #pragma unroll
        for (int d = 0; d < DTH; d++) o[t][d] = scaled(o[t][d], factor);
      }
      if (t == 0) few_values<0>(value_at(Few::at(buf, 1), l16, lq) + (kg * CG + (dt0 >> 1)) * 1024, vt);
      if (odd) add_odd<DTH>(st, odd, t0, lo[t] - t0, hi[t] - t0, o[t], dt0, lq);
      #pragma unroll
      for (int k = 0; k < FEW_TERMS; k++) {
        const s16x4 p = __builtin_bit_cast(s16x4, pack(s[0]));
        sum[t] = mma16(ones, p, sum[t]);
        #pragma unroll
        for (int d = 0; d < DTH; d++) o[t][d] = mma16(vt[d], p, o[t][d]);
      }
    }
    buf = buf == Few::ST - 1 ? 0 : buf + 1;
  }
  bool bad = false;
  #pragma unroll
  for (int t = 0; t < RT; t++) bad |= not_finite(o[t], sum[t]);
  if (bad && !careful) lds.not_finite = 1;
  // the key groups meet: maxima and sums, then the outputs, group after group
  __syncthreads();
  if (!careful && __builtin_amdgcn_readfirstlane(lds.not_finite)) return true;
  float* stat = (float*)lds.pages;                       // [2][KG][16·RT], by the waves of the first dims
  float* acc = (float*)lds.ring;                         // [KG][16·RT][HD]
  if (dh == 0 && lq == 0) {
    #pragma unroll
    for (int t = 0; t < RT; t++) stat[kg * 32 + t * 16 + l16] = m[t], stat[128 + kg * 32 + t * 16 + l16] = sum[t][0];
  }
  __syncthreads();
  #pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = t * 16 + l16;
    float mx = NEG_INF;
    for (int k = 0; k < KG; k++) mx = __builtin_fmaxf(mx, stat[k * 32 + row]);
    const float f = mx == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m[t] - mx);
    #pragma unroll
    for (int d = 0; d < DTH; d++)
      if (dt0 + d < DT) *(f32x4*)&acc[(kg * 16 * RT + row) * HD + (dt0 + d) * 16 + lq * 4] = careful ? scaled(o[t][d], f) : o[t][d] * f;
  }
  __syncthreads();
  for (int u = tid; u < it.rows * (HD / 4); u += 256) {
    const int row = u / (HD / 4), d = u % (HD / 4) * 4;
    float mx = NEG_INF, l = 0.0f;
    for (int k = 0; k < KG; k++) mx = __builtin_fmaxf(mx, stat[k * 32 + row]);
    // (scores that are all NaN leave no maximum, and sums of NaN)
    for (int k = 0; k < KG; k++) l += stat[128 + k * 32 + row] * (mx == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(stat[k * 32 + row] - mx));
    f32x4 v = *(const f32x4*)&acc[row * HD + d];
    for (int k = 1; k < KG; k++) v += *(const f32x4*)&acc[(k * 16 * RT + row) * HD + d];
    if (it.splits == 1) {
      put4(a.o + out_at(it, g, row) + d, l == 0.0f ? (f32x4){0, 0, 0, 0} : v / l);
    } else {
      const int at = it.slot + (it.split ? it.split * 2 * stride : stride) + row;
      *(f32x4*)(part_sums(a, g, at) + d) = v;
      if (d == 0) {
        float* p = part_stats(a, g, at);
        p[0] = mx, p[1] = l;
      }
    }
  }
  if (it.splits > 1) meet(a, it, g, 0, it.rows, 2 * stride, stride);
  return false;
}

// Oᵀ += Vᵀ·P over the tile, eight reads (all keys of two or four tiles of dims) at a time
template <int D>
__device__ __forceinline__ void many_values(unsigned at, const s16x8 (&p)[2][MANY_TK / 32][MANY_TERMS], f32x4 (&o)[2][DT]) {
  constexpr int KS = MANY_TK / 32, G = 8 / (MANY_TK / 16);    // dim tiles a group
  constexpr int B0 = D / 2, B1 = D / 2 + 1 < CG ? D / 2 + 1 : D / 2;
  s16x4 r[8];
  if constexpr (KS == 2) tr_read8<B0 * 1024, (CG + B0) * 1024, (2 * CG + B0) * 1024, (3 * CG + B0) * 1024>(at, r);
  else tr_read8<B0 * 1024, (CG + B0) * 1024, B1 * 1024, (CG + B1) * 1024>(at, r);
  #pragma unroll
  for (int e = 0; e < G; e++) {
    if (D + e >= DT) break;
    #pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const int i = KS == 2 ? 4 * ks + e : 4 * (e / 2) + e % 2;
      const s16x8 v = __builtin_shufflevector(r[i], r[i + 2], 0, 1, 2, 3, 4, 5, 6, 7);
      #pragma unroll
      for (int k = 0; k < MANY_TERMS; k++) {
        o[0][D + e] = mma32(v, p[0][ks][k], o[0][D + e]);
        o[1][D + e] = mma32(v, p[1][ks][k], o[1][D + e]);
      }
    }
  }
  if constexpr (D + G < DT) many_values<D + G>(at, p, o);
}

// ── many rows: 32 a wave ──────────────────────────────────────────────────────────────────────────
__device__ __forceinline__ bool many_rows(const Args& a, const Item& it, int g, Stream& st, int t_first, int t_last, int lo_all, int hi_all, int full_lo, int full_hi, bool careful) {
  constexpr int TK = MANY_TK, NK = TK / 16;
  const int tid = st.tid, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lq = lane >> 4;
  const int row0 = it.tile * PR + wave * 32;
  s16x8 qf[2][DSTEP];
  int lo[2], hi[2];
  #pragma unroll
  for (int t = 0; t < 2; t++) {
    int row = row0 + t * 16 + l16;
    if (row >= it.rows) row = it.rows - 1;
    const unsigned short* q = a.q + (QB + (it.start + row / REP) * Q0 + (g * REP + row % REP) * Q1);
    read_row(q, lq, qf[t]);
    hi[t] = clamp_pos(it.past + row / REP + 1);
    lo[t] = W ? clamp_pos(it.past + row / REP + 1 - W) : 0;
  }
  // this wave's rows: what any and what all of them see
  const int first = row0 < it.rows ? row0 : it.rows - 1, last = row0 + 31 < it.rows ? row0 + 31 : it.rows - 1;
  const int wave_hi = clamp_pos(it.past + last / REP + 1), all_hi = clamp_pos(it.past + first / REP + 1);
  const int wave_lo = W ? clamp_pos(it.past + first / REP + 1 - W) : 0, all_lo = W ? clamp_pos(it.past + last / REP + 1 - W) : 0;
  const bool idle = row0 >= it.rows;
  f32x4 o[2][DT], sum[2];
  float m[2];
  #pragma unroll
  for (int t = 0; t < 2; t++) {
    m[t] = NEG_INF, sum[t] = (f32x4){0, 0, 0, 0};
    #pragma unroll
    for (int d = 0; d < DT; d++) o[t][d] = (f32x4){0, 0, 0, 0};
  }
  begin<Many>(st, t_first, t_last, qf);
  const short one = HALF ? (short)0x3C00 : (short)0x3F80;
  const s16x8 ones = {one, one, one, one, one, one, one, one};
  int buf = 0;
  for (int i = t_first; i < t_last; i++) {
    const int t0 = i * TK;
    turn<Many>(st, i, t_last, buf);
    const unsigned long long holes = lds.holes ? st.missing<TK>(t0) : 0;
    unsigned long long odd = 0;
    if (!(t0 >= full_lo && t0 + TK <= full_hi) || holes || careful) {
      // the tile is every wave's: cleaned by all, then used
      if (tid == 0) lds.odd_keys = 0;
      __syncthreads();
      const unsigned long long mine = clean(Many::at(buf, 1), holes, 0, TK, 0, CH, lo_all - t0, hi_all - t0, tid, 256);
      if (mine) atomicOr(&lds.odd_keys, mine);
      __syncthreads();
      odd = lds.odd_keys;
    }
    if (!idle && t0 < wave_hi && t0 + TK > wave_lo) {
      const bool full = !careful && t0 >= all_lo && t0 + TK <= all_hi && !holes;
      f32x4 s[2][NK];
      #pragma unroll
      for (int kt = 0; kt < NK; kt++) {
        s[0][kt] = (f32x4){0, 0, 0, 0}, s[1][kt] = (f32x4){0, 0, 0, 0};
        #pragma unroll
        for (int d = 0; d < DSTEP; d++) {
          const s16x8 k = key_run(Many::at(buf, 0), kt, d, l16, lq);
          s[0][kt] = mma32(k, qf[0][d], s[0][kt]);
          s[1][kt] = mma32(k, qf[1][d], s[1][kt]);
        }
      }
      s16x8 p[2][NK / 2][MANY_TERMS];
      #pragma unroll
      for (int t = 0; t < 2; t++) {
        float factor;
        weigh<NK>(s[t], full, holes, lq * 4, lo[t] - t0, hi[t] - t0, careful ? 0.0f : 8.0f, m[t], factor);
        if (!__all(factor == 1.0f)) {
          sum[t] *= factor;
          #pragma unroll
          for (int d = 0; d < DT; d++) o[t][d] = scaled(o[t][d], factor);
        }
        if (odd) add_odd<DT>(st, odd, t0, lo[t] - t0, hi[t] - t0, o[t], 0, lq);
        #pragma unroll
        for (int ks = 0; ks < NK / 2; ks++)
          #pragma unroll
          for (int k = 0; k < MANY_TERMS; k++) {
            const u32x2 x = pack(s[t][2 * ks]), y = pack(s[t][2 * ks + 1]);
            p[t][ks][k] = __builtin_bit_cast(s16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3));
            sum[t] = mma32(ones, p[t][ks][k], sum[t]);
          }
      }
      many_values<0>(value_at(Many::at(buf, 1), l16, lq), p, o);
    }
    buf = buf == Many::ST - 1 ? 0 : buf + 1;
  }
  if (!careful && (not_finite(o[0], sum[0]) || not_finite(o[1], sum[1]))) lds.not_finite = 1;
  __syncthreads();
  if (!careful && __builtin_amdgcn_readfirstlane(lds.not_finite)) return true;
  const int tile_rows = it.rows - it.tile * PR < PR ? it.rows - it.tile * PR : PR;
  #pragma unroll
  for (int t = 0; t < 2; t++) {
    const int r = wave * 32 + t * 16 + l16;
    if (r >= tile_rows) continue;
    const float l = sum[t][0];
    if (it.splits == 1) {
      const float f = l == 0.0f ? 0.0f : 1.0f / l;
      #pragma unroll
      for (int d = 0; d < DT; d++) put4(a.o + out_at(it, g, it.tile * PR + r) + d * 16 + lq * 4, o[t][d] * f);
    } else {
      float* p = part_sums(a, g, it.slot + it.split * PR + r);
      #pragma unroll
      for (int d = 0; d < DT; d++) *(f32x4*)(p + d * 16 + lq * 4) = o[t][d];
      if (lq == 0) {
        float* x = part_stats(a, g, it.slot + it.split * PR + r);
        x[0] = m[t], x[1] = l;
      }
    }
  }
  if (it.splits > 1) meet(a, it, g, it.tile * PR, tile_rows, PR, 0);
  return false;
}

// Rows [r0, r1) of an item: what any and what all of them see, and the part of the key tiles. True where
// a sum came out not finite: nothing has been stored then, and the rows are taken again, with `careful`
// (from here, not inside: what a second pass keeps in registers would cost the first one its own).
template <bool MANY>
__device__ __forceinline__ bool rows_of(const Args& a, const Item& it, int g, int r0, int r1, int t0, int t1, int stride, bool careful) {
  constexpr int TK = MANY ? MANY_TK : FEW_TK;
  const long long p0 = it.past + r0 / REP, p1 = it.past + (r1 - 1) / REP;
  const int hi_all = clamp_pos(p1 + 1), full_hi = clamp_pos(p0 + 1);
  const int lo_all = W ? clamp_pos(p0 + 1 - W) : 0, full_lo = W ? clamp_pos(p1 + 1 - W) : 0;
  const int k0 = lo_all / TK, k1 = lo_all < hi_all ? (hi_all + TK - 1) / TK : k0;
  // (an opaque copy, so that nothing a lane computes from it is kept in registers around a second pass)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  Stream st{a, a.tables + (long long)it.b * M, tid, g, lo_all / BS, (hi_all - 1) / BS, 0, a.k + (KB + g * K1), a.v + (VB + g * V1)};
  if constexpr (MANY) {
    const int t_first = k0 + (int)((long long)(k1 - k0) * it.split / it.splits), t_last = k0 + (int)((long long)(k1 - k0) * (it.split + 1) / it.splits);
    return many_rows(a, it, g, st, t_first, t_last, lo_all, hi_all, full_lo, full_hi, careful);
  } else {
    const int t_first = k0 + t0 < k1 ? k0 + t0 : k1, t_last = k0 + t1 < k1 ? k0 + t1 : k1;
    if (it.rows <= 16) return few_rows<1>(a, it, stride, g, st, t_first, t_last, lo_all, hi_all, full_lo, full_hi, careful);
    return few_rows<2>(a, it, stride, g, st, t_first, t_last, lo_all, hi_all, full_lo, full_hi, careful);
  }
}

extern "C" __global__ void __launch_bounds__(256, OCC) sanic_paged_attn(Args a) {
  const int g = (int)(blockIdx.x % NKV), lane = threadIdx.x & 63;
  int w = (int)(blockIdx.x / NKV);
  Req q;
  const Plan p = make_plan(a, q);
  // (a run outside the grid would leave its request's arrivals part-counted, for later launches to find)
  if (p.none) return;
  Item it;
  // the many-row items first: they take longest
  if (PITEMS && w < p.items) {
    find_many(a, p, q, w, it);
    const int r0 = it.tile * PR, r1 = r0 + PR < it.rows ? r0 + PR : it.rows;
    for (bool careful = false; rows_of<true>(a, it, g, r0, r1, 0, 0, 0, careful); careful = true) __syncthreads();
    return;
  }
  // the requests in the w-th run of key tiles
  w -= p.items;
  const int r0 = w * p.run, r1 = r0 + p.run;
  int before = 0;
  for (int b0 = 0; b0 < B && before < r1; b0 += 64) {
    if (B > 64) q = request(a, b0 + lane);
    const int mine = q.tiles == 0 && q.rows ? q.kt : 0, inc = before + scan64(mine), exc = inc - mine;
    unsigned long long who = __ballot(mine > 0 && inc > r0 && exc < r1);
    while (who) {
      const int l = __builtin_ctzll(who), from = pick(exc, l), to = pick(inc, l), w0 = from / p.run;
      who &= who - 1;
      it.b = b0 + l, it.tile = -1, it.rows = pick(q.rows, l);
      it.splits = (to - 1) / p.run - w0 + 1, it.split = w - w0;
      it.slot = w0 * 2 * p.stride;             // a request's first part is its workgroup's second partial
      it.count = it.b;
      it.start = pick(q.start, l), it.past = pick(q.past, l);
      const int t0 = (r0 > from ? r0 : from) - from, t1 = (r1 < to ? r1 : to) - from;
      for (bool careful = false; rows_of<false>(a, it, g, 0, it.rows, t0, t1, p.stride, careful); careful = true) __syncthreads();
      __syncthreads();
    }
    before = pick(inc, 63);
  }
}
)SRC";

// The matrix-core kernel takes queries and caches of one 16-bit type whose rows are runs of a multiple
// of 16 elements, in units of 16 bytes.
static bool mfma_takes(const OperandView& q, const OperandView& k, const OperandView& v, int64_t B, int64_t M) {
    const int64_t HD = q.extent[2];
    if (q.dtype != k.dtype || (q.dtype != SANIC_BF16 && q.dtype != SANIC_F16) || HD % 16 || HD > 256) return false;
    if (B * (M * k.extent[2] / 32 + 1) >= int64_t(1) << 30) return false;     // key tiles are counted in 31 bits
    for (const OperandView* o : {&k, &v})
        if (o->stride[2] < 0 || o->stride[2] >= int64_t(1) << 26) return false;   // 16 rows of a page: an unsigned offset of 32 bits
    for (const OperandView* o : {&q, &k, &v}) {
        if (o->stride.back() != 1 || o->base % 8) return false;
        for (size_t j = 0; j + 1 < o->stride.size(); j++)
            if (o->stride[j] % 8) return false;
    }
    return true;
}

LoweredStage lower_paged_attn(const sanic_program_desc* d, const sanic_stage& st, int64_t& scratch) {
    OperandView q, k, v;
    operand_view(d, st.leaf[0], q), operand_view(d, st.leaf[1], k), operand_view(d, st.leaf[2], v);
    const int64_t T = q.extent[0], NH = q.extent[1], HD = q.extent[2], NB = k.extent[0], NKV = k.extent[1], BS = k.extent[2];
    const sanic_node& tables = d->nodes[st.leaf[3]];
    const int64_t B = tables.shape[0], M = tables.shape[1], REP = NH / NKV;
    const double scale = d->nodes[st.leaf[6]].value;
    std::string c;
    auto number = [](const char* n, int64_t v) { return std::string("constexpr int ") + n + " = " + std::to_string(v) + ";\n"; };
    c += number("T", T) + number("NH", NH) + number("HD", HD) + constant("NB", NB) + number("BS", BS) + number("REP", REP);
    c += number("B", B) + number("M", M) + constant("W", st.stream) + number("NKV", NKV);
    c += constant("DQ", q.dtype) + constant("DC", k.dtype) + constant("DO", st.out_dtype) + "constexpr float SCALE = " + flit(scale) + ";\n";
    auto strides = [&](const char* n, const OperandView& o) {
        for (size_t j = 0; j < o.stride.size(); j++) c += constant((std::string(n) + std::to_string(j)).c_str(), o.stride[j]);
        c += constant((std::string(n) + "B").c_str(), o.base);
    };
    strides("Q", q), strides("K", k), strides("V", v);
    LoweredStage L;
    Launch ln{"sanic_paged_attn", "", dim3((unsigned)((T * NH + 3) / 4)), dim3(256), 0, {}};
    for (int b : {q.buffer, k.buffer, v.buffer, tables.buffer, d->nodes[st.leaf[4]].buffer, d->nodes[st.leaf[5]].buffer, st.out_buffer})
        ln.args.push_back({Arg::BUF, b});
    // Tiles and rings: what lets OCC workgroups share 160 KB of LDS and, at 256 threads, 512 / OCC
    // registers. Heads of 64: tiles of 64 keys, 3 deep, 3 workgroups a CU (24 requests of 5 drafts 49.8
    // us, a mixed batch 60.8; with the plan of that time 55.8 and 63.2 against 63.8 and 73.3 for tiles
    // of 32 and 4 workgroups, 63.5 and 77.5 for 2 workgroups). Heads of 128: 2 workgroups, many rows in
    // tiles of 64 in a ring of 2 (those 4096 rows 1660 us at that time; tiles of 32 in a ring of 3
    // 1770). Few-row workgroups as many as are resident: 2/3 of them 63.9 us for the drafts, twice as
    // many 68.7, against 55.8. Heads of 160 to 256: a decode batch of 64 over up to 4000 tokens, 24 requests
    // of 5 drafts over up to 3000, and 2048 rows behind 4096 tokens, us with 1 and with 2 workgroups a CU:
    // 160 275 and 168, 132 and 117, 703 and 351; 192 286 and 182, 143 and 134, 743 and 376; 256 355 and 259,
    // 219 and 204, 880 and 483. Rings of 3 instead of 2 are the same within 2% for all of these.
    const int64_t FEW_TK = HD <= 64 ? 64 : 32, FEW_ST = HD <= 64 ? 3 : HD <= 128 ? 4 : 2;
    const int64_t MANY_TK = HD <= 128 ? 64 : 32, MANY_ST = HD <= 64 ? 3 : 2, OCC = HD <= 64 ? 3 : 2;
    const int64_t PR = 128, DR = 32, MOST = 256, LINE = 16;
    const int64_t slots = 256 * OCC;
    const int64_t live = std::min(B, T), groups = std::max<int64_t>(1, slots / NKV);
    const int64_t budget = partial_room() / (NKV * (HD + 2) * 4);
    const int64_t DROWS = std::min(2 * groups * std::min(DR, (T * REP + LINE - 1) / LINE * LINE), std::max(budget, 2 * DR)) / LINE * LINE;
    const int64_t tiles = T * REP > DR ? T * REP / PR + std::min(live, T * REP / (DR + 1)) : 0;
    const int64_t PSPLIT = tiles ? std::min(2 * slots / NKV, budget / PR) : 0;
    const int64_t SLOTS = DROWS + PSPLIT * PR, per_head = groups + std::max(tiles, PSPLIT);
    // a workgroup's first key tile, its number times the run's length, stays within 31 bits
    const int64_t most = M * BS / FEW_TK + 2, fit = std::max<int64_t>(1, std::min(groups, DROWS / (2 * DR)));
    const double run = 1.002 * std::max((double)B * most / fit, (double)most / MOST) + 2;
    // arrival counters: a head's on lines of their own (a line that several XCDs count on goes back and
    // forth between them), each on one while the 16384 static ones last
    int64_t cpad = 32;
    auto counts = [&] { return ((B + PSPLIT / 2 + 1) * cpad + 31) / 32 * 32; };
    while (cpad > 1 && counts() * NKV > 16384) cpad /= 2;
    // two parts a key head of very many key heads, or their counters, would pass the static scratch
    const bool room = NKV * (SLOTS * (HD + 2) + counts()) * 4 <= 2 * kPartialRoom + (int64_t(1) << 20);
    if (!mfma_takes(q, k, v, B, M) || !std::isfinite(scale) || (per_head + 1) * run >= 2147483648.0 || !room) {
        L.kernel_kind = "operator:paged_attn[plain]";
        L.source = std::string(kPrelude) + kElement + c + kPlain;
        L.launches.push_back(ln);
        return L;
    }
    c += number("FEW_TK", FEW_TK) + number("FEW_ST", FEW_ST) + number("MANY_TK", MANY_TK) + number("MANY_ST", MANY_ST);
    c += number("OCC", OCC) + number("PR", PR) + number("DR", DR) + number("MOST", MOST) + number("LINE", LINE);
    c += number("FEW_GROUPS", groups) + number("DROWS", DROWS) + number("PITEMS", tiles > 0) + number("PSPLIT", PSPLIT) + number("SLOTS", SLOTS);
    c += number("COUNTS", counts()) + number("CPAD", cpad);
    c += number("ONE_XCD", xcd_local_enabled() && NKV % 8 == 0);
    c += number("PAGES", 512) + number("FLIP", scale < 0) + "constexpr float C2 = " + flit(std::fabs(scale) * 1.4426950408889634) + ";\n";
    // Weights take the 16 bits of the matrix cores' operands. Few rows are bound by the cache's bytes: a
    // second term (what the rounding left) costs nothing there. Many rows are bound by the products and
    // keep one term where the output is 16 bits too: half a step of relative error a weight, of both signs,
    // in sums divided by the same rounded weights' sum (RMS error against 64 bits, bf16, 2.3e-3; with two
    // terms 1.7e-3, the output's own rounding, at 1499 us instead of 1186 for 4096 rows of heads of 128
    // behind 12288 tokens, and 71.5 instead of 55.6 for a mixed batch of heads of 64). A caller that wants
    // more asks for an f32 output: 24 bits from three terms (f16: 22 from two, and the rest; RMS 9e-8).
    c += number("FEW_TERMS", st.out_dtype == SANIC_F32 ? 3 : 2) + number("MANY_TERMS", st.out_dtype == SANIC_F32 ? 3 : 1);
    L.kernel_kind = "operator:paged_attn[mfma]";
    L.source = std::string(kPrelude) + kElement + c + kMfma;
    ln.grid = dim3((unsigned)(NKV * per_head));
    ln.args.push_back({Arg::SCRATCH, shared_scratch(scratch, NKV * SLOTS * (HD + 2) * 4)});
    ln.args.push_back({Arg::COUNTERS, shared_counters(counts() * NKV)});
    L.launches.push_back(ln);
    return L;
}

}  // namespace sanic
