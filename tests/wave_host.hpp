// Runs a generated kernel on the CPU, one workgroup after the other: every lane is a fiber, the 64
// lanes of a wave meet at each cross-lane operation, the workgroup at each barrier. Buffers lie
// between pages that cannot be touched, loads into LDS land only when the kernel waits for them.
// The kernel's text stands between this file and wave_host_main.hpp.
#include <math.h>
#include <signal.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <unistd.h>

#include <vector>

#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

typedef long long idx_t;

namespace wh {

struct Dim { unsigned x; };
struct Load { char* to; char bytes[16]; };
struct Lane {
  Dim thread;
  void* sp;
  bool done;
  std::vector<Load> under_way;     // loads into LDS, oldest first
};
struct Wave {
  unsigned count = 0, gen = 0;
  int what[2][64];
  alignas(16) char in[2][64][48];
};
static Lane lanes[256];
static Wave waves[4];
static Lane* me;
static Dim block, grid;
static void* scheduler;
static unsigned live, at_barrier, barrier_gen;
static unsigned long long progress;
static const char *ring_lo, *ring_hi;

[[noreturn]] static void stop(const char* why) {
  fprintf(stderr, "workgroup %u thread %u: %s\n", block.x, me ? me->thread.x : 0, why);
  fflush(stderr);
  _exit(3);
}

extern "C" void wh_swap(void** from, void* to);
asm(R"(
.text
.type wh_swap,@function
wh_swap:
  pushq %rbp
  pushq %rbx
  pushq %r12
  pushq %r13
  pushq %r14
  pushq %r15
  movq %rsp, (%rdi)
  movq %rsi, %rsp
  popq %r15
  popq %r14
  popq %r13
  popq %r12
  popq %rbx
  popq %rbp
  ret
)");
__attribute__((noinline)) static void yield() { wh_swap(&me->sp, scheduler); }

static void land(size_t left) {
  auto& q = me->under_way;
  size_t n = q.size() > left ? q.size() - left : 0;
  for (size_t i = 0; i < n; i++) memcpy(q[i].to, q[i].bytes, 16);
  q.erase(q.begin(), q.begin() + n);
}

// every lane of the wave brings `n` bytes to operation `what`; all of them come back
static const char (*exchange(int what, const void* p, size_t n))[48] {
  const unsigned lane = me->thread.x & 63;
  Wave& w = waves[me->thread.x >> 6];
  const unsigned g = w.gen, s = g & 1;
  memcpy(w.in[s][lane], p, n);
  w.what[s][lane] = what;
  if (++w.count == 64) {
    for (int i = 0; i < 64; i++)
      if (w.what[s][i] != what) stop("lanes of a wave meet at different operations");
    w.count = 0;
    w.gen++;
    progress++;
  } else {
    while (w.gen == g) yield();
  }
  return w.in[s];
}
template <class T> static T get(const char (*in)[48], unsigned lane) {
  T v;
  memcpy(&v, in[lane], sizeof(T));
  return v;
}
static void wave_sync() { char c = 0; exchange(1, &c, 1); }
static void barrier() {
  land(0);
  const unsigned g = barrier_gen;
  if (++at_barrier == live) {
    at_barrier = 0;
    barrier_gen++;
    progress++;
  } else {
    while (barrier_gen == g) yield();
  }
}
static void turn_barrier(size_t left) {   // s_waitcnt vmcnt(left); s_barrier
  land(left);
  const unsigned g = barrier_gen;
  if (++at_barrier == live) {
    at_barrier = 0;
    barrier_gen++;
    progress++;
  } else {
    while (barrier_gen == g) yield();
  }
}
static int barrier_or(int x) {
  static int any[2];
  const unsigned s = barrier_gen & 1;
  if (x) any[s] = 1;
  barrier();
  const int out = any[s];
  barrier();
  any[s] = 0;
  barrier();
  return out;
}
template <class T> static T shfl(int what, T v, unsigned lane) { return get<T>(exchange(what, &v, sizeof v), lane); }
template <class T> static T shfl_up(T v, unsigned o) {
  const unsigned l = me->thread.x & 63;
  return shfl(2, v, l >= o ? l - o : l);
}
template <class T> static T shfl_xor(T v, unsigned o) { return shfl(3, v, (me->thread.x & 63) ^ o); }
static unsigned long long ballot(bool v) {
  auto in = exchange(4, &v, 1);
  unsigned long long out = 0;
  for (int i = 0; i < 64; i++) out |= (unsigned long long)(in[i][0] != 0) << i;
  return out;
}
static int readlane(int v, unsigned lane) {
  if (lane > 63) stop("readlane of a lane past 63");
  return shfl(5, v, lane);
}
static int readfirst(int v) { return shfl(6, v, 0); }
template <class F> static float reduce(int what, float v, F f, int step) {   // over lanes equal mod `step`
  auto in = exchange(what, &v, 4);
  float out = get<float>(in, me->thread.x % step);
  for (int i = me->thread.x % step + step; i < 64; i += step) out = f(out, get<float>(in, i));
  return out;
}
static void load_lds(const void* from, void* to, int bytes, int offset) {
  struct { void* to; } base{to};
  auto in = exchange(7, &base, sizeof base);
  for (int i = 0; i < 64; i++)
    if (get<void*>(in, i) != to) stop("a load into LDS whose base differs between lanes");
  Load l;
  l.to = (char*)to + offset + (me->thread.x & 63) * 16;
  if (bytes != 16 || l.to < ring_lo || l.to + 16 > ring_hi) stop("a load into LDS outside its ring");
  memcpy(l.bytes, from, 16);
  me->under_way.push_back(l);
}
// 16 lanes read 4 elements each, and lane i gets element i % 4 of lanes i / 4, i / 4 + 4, ...
template <class V> static void transposed(unsigned at, V& out) {
  const char* p = (const char*)(size_t)at;
  if (p < ring_lo || p + 8 > ring_hi) stop("a transposed read outside the ring");
  char x[8];
  memcpy(x, p, 8);
  auto in = exchange(8, x, 8);
  const unsigned l = me->thread.x & 63, first = l & ~15u, i = l & 15;
  short e[4];
  for (int j = 0; j < 4; j++) memcpy(&e[j], in[first + j * 4 + i / 4] + (i % 4) * 2, 2);
  memcpy(&out, e, 8);
}
static float as_float(unsigned u) { float f; memcpy(&f, &u, 4); return f; }
static unsigned as_uint(float f) { unsigned u; memcpy(&u, &f, 4); return u; }
static float widen(short s, bool half) {
  if (!half) return as_float((unsigned)(unsigned short)s << 16);
  _Float16 h;
  memcpy(&h, &s, 2);
  return (float)h;
}
// D[4·(lane / 16) + r][lane % 16] += Σ A[row][k]·B[k][col]; a lane holds PER of k from PER·(lane / 16) on
template <int PER, bool HALF, class X, class C> static C product(const X& a, const X& b, C c) {
  struct { short a[PER], b[PER]; } v;
  static_assert(sizeof(X) == 2 * PER);
  memcpy(v.a, &a, 2 * PER);
  memcpy(v.b, &b, 2 * PER);
  auto in = exchange(9 + PER, &v, sizeof v);
#ifndef WH_NO_MATH
  const int l = me->thread.x & 63, col = l & 15, row0 = l / 16 * 4;
  float y[4 * PER];
  for (int q = 0; q < 4; q++)
    for (int k = 0; k < PER; k++) y[q * PER + k] = widen(((const short*)in[q * 16 + col])[PER + k], HALF);
  for (int r = 0; r < 4; r++) {
    double sum = c[r];
    for (int q = 0; q < 4; q++)
      for (int k = 0; k < PER; k++) sum += (double)widen(((const short*)in[q * 16 + row0 + r])[k], HALF) * y[q * PER + k];
    c[r] = (float)sum;
  }
#endif
  return c;
}
static float exp2_flushed(float x) {
  const float e = exp2f(x);
  return e < 0x1p-126f ? 0.0f : e;
}

}  // namespace wh

#define threadIdx (wh::me->thread)
#define blockIdx (wh::block)
#define gridDim (wh::grid)
#define __syncthreads() wh::barrier()
#define __syncthreads_or(x) wh::barrier_or(x)
#define __shfl_up(v, o) wh::shfl_up(v, o)
#define __shfl_xor(v, o) wh::shfl_xor(v, o)
#define __ballot(p) wh::ballot(p)
#define __all(p) (wh::ballot(p) == ~0ull)
#define __any(p) (wh::ballot(p) != 0)
#define __uint_as_float(u) wh::as_float(u)
#define __float_as_uint(f) wh::as_uint(f)
#define __expf(x) expf(x)
#define __builtin_amdgcn_readlane(v, l) wh::readlane(v, l)
#define __builtin_amdgcn_readfirstlane(v) wh::readfirst(v)
#define __builtin_amdgcn_exp2f(x) wh::exp2_flushed(x)
#define __builtin_amdgcn_s_waitcnt(n) wh::land(0)
#define __builtin_amdgcn_fence(order, scope) (strcmp(scope, "wavefront") ? (void)0 : wh::wave_sync())
#define __builtin_amdgcn_global_load_lds(from, to, bytes, offset, aux) wh::load_lds((const void*)(from), (void*)(to), bytes, offset)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) wh::product<8, true>(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) wh::product<8, false>(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, x, y, z) wh::product<4, true>(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, x, y, z) wh::product<4, false>(a, b, c)
#define __HIP_MEMORY_SCOPE_AGENT 0
template <class T> static T wh_add(T* p, T v) { const T old = *p; *p += v; return old; }
#define __hip_atomic_fetch_add(p, v, order, scope) wh_add(p, v)
template <class T> static T atomicOr(T* p, T v) { const T old = *p; *p |= v; return old; }
template <class T> static T atomicMin(T* p, T v) { const T old = *p; if (v < old) *p = v; return old; }
template <class T> static T atomicMax(T* p, T v) { const T old = *p; if (v > old) *p = v; return old; }

static float sanic_bf16(unsigned short b) { return wh::as_float((unsigned)b << 16); }
static unsigned short sanic_to_bf16(float v) {
  const unsigned b = wh::as_uint(v);
  if (v != v) return (unsigned short)(b >> 16 | 0x40u);
  return (unsigned short)((b + 0x7FFFu + (b >> 16 & 1u)) >> 16);
}
extern "C" __bf16 __truncsfbf2(float v) {
  const unsigned short b = sanic_to_bf16(v);
  __bf16 out;
  memcpy(&out, &b, 2);
  return out;
}
static float wh_plus(float x, float y) { return x + y; }
static float wh_most(float x, float y) { return __builtin_fmaxf(x, y); }
static float sanic_wave_sum(float v) { return wh::reduce(30, v, wh_plus, 1); }
static float sanic_wave_max(float v) { return wh::reduce(31, v, wh_most, 1); }
static float sanic_rows_sum(float v) { return wh::reduce(32, v, wh_plus, 16); }
static float sanic_rows_max(float v) { return wh::reduce(33, v, wh_most, 16); }
