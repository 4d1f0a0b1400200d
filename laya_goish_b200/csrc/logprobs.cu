// Log probabilities of given tokens, entropy and the likeliest tokens of
// full-vocabulary logit rows, each row read once.
//
// With any reference M near the row's maximum and c = fl(M log2 e),
//   y = fl(x log2 e - c) (one FMA),  s = sum 2^y,  a = sum 2^y y,
//   lse = c ln 2 + ln s,  logprob_j = y_j ln 2 - ln s,  entropy = ln s - ln 2 a / s.
// c's own rounding is the same in every term and cancels; y has one rounding,
// relative to y itself.  (From |M| = 65000 on, y = fl((x - M) log2 e), and M
// takes the place of c ln 2.)  Every thread keeps its own (M, s, a) and moves M only
// when a value passes it by more than 6 (terms of up to e^6 cost no precision in
// F32), so the rescale is rare; the threads' states are merged at the end.
//
// The `top` best come from the same pass: the row is cut into contiguous
// segments and the pass leaves each segment's maximum in shared memory.
// Order elements by (value descending, index ascending) and segments by
// (maximum descending, index ascending): an element outside the best `top`
// segments is preceded by the maxima of `top` segments, so the best `top`
// elements lie in the best `top` segments, ties included, whatever the row
// holds.  Only those segments are read again (from L2): elements from the
// last chosen segment's maximum t on go to a list that is ranked.  Where it
// overflows (many equal to t), those beyond t are listed and the first equal
// to t follow in index order.
//
// Bound by HBM (the row's bytes), with two others close behind for 16-bit rows:
// one exponential per element (16 per SM and clock) and the issue slots, which
// is why the arithmetic runs on packed pairs and a vector's maximum and minimum
// are taken before it is widened.
#include <algorithm>
#include <atomic>

#include "device_ops.h"
#include "launch.h"
#include "ptx.cuh"

namespace laya {

namespace {

constexpr int kMaxSeg = 512;   // segments per row
constexpr int kCand = 1024;    // list of the best elements
constexpr int kChunk = 1024;   // 16-byte vectors per ring stage
constexpr int kRingWarps = 8;  // consumer warps of the ring form
constexpr int kMaxStages = 8;
constexpr long long kBudget = 400000000ll;  // SM cycles per bounded wait (~0.2 s)

struct LpArgs {
  const void* x;
  long long stride;  // elements
  int rows, vocab;
  const int* tokens;
  long long tstride;
  int n_tok, top;
  float* lp;
  float* ent;
  float* lse;
  int* ids;
  float* tlp;
  unsigned* status;
  int seg_vec;  // vectors per segment, a power of two
  int stages;   // ring stages (0: rows read straight into registers)
};

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 6.f;
// References for which y = fl(x log2 e - c), with c = fl(M log2 e) off by less
// than 2^-7.  Farther out that error grows past what 2^y can hold (half an ulp
// of M log2 e is 512 at 1e10), and y = fl((x - M) log2 e) instead: so is a row
// of masked tokens alone (-1e10, the type's lowest value) or of large logits.
constexpr float kNear = 65000.f;
__device__ __forceinline__ bool near(float M) { return fabsf(M) < kNear; }
// Stands for smaller values of F32 and BF16 at a near reference: e^(x - M) is 0.
constexpr float kFloor = -1e30f;

// u32 of the same order; -0 counts as +0
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kNegInfKey = 0x007fffffu;  // order_key(-inf)

// 16-byte pieces of a row.  top: the maximum of several (NaNs left out); it and
// the bound are taken on packed pairs, before widening.  unpack: the values in
// F32; BOUND: no less than a finite bound (a NaN stays), at which e^(x - M) is 0
// for every near reference M: -65504 for F16, 504 below the lowest of them.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(float x) { return x; }
  template <int NV>
  static __device__ __forceinline__ float top(const uint4 (&w)[NV]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; i++)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(w[i].x), __uint_as_float(w[i].y)),
                         fmaxf(__uint_as_float(w[i].z), __uint_as_float(w[i].w))));
    return m;
  }
  template <bool BOUND>
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = BOUND ? max_nan(__uint_as_float(w[i]), kFloor) : __uint_as_float(w[i]);
  }
};
template <>
struct Elem<half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(half x) { return __half2float(x); }
  template <int NV>
  static __device__ __forceinline__ float top(const uint4 (&w)[NV]) {
    const half2* h = reinterpret_cast<const half2*>(w);
    half2 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * NV; i++) m = __hmax2(m, h[i]);
    return fmaxf(__low2float(m), __high2float(m));
  }
  template <bool BOUND>
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[8]) {
    const half2* h = reinterpret_cast<const half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(BOUND ? __hmax2_nan(h[i], __float2half2_rn(-65504.f)) : h[i]);
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  template <int NV>
  static __device__ __forceinline__ float top(const uint4 (&w)[NV]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    __nv_bfloat162 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * NV; i++) m = __hmax2(m, h[i]);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
    return fmaxf(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  template <bool BOUND>
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 x = BOUND ? __hmax2_nan(h[i], __float2bfloat162_rn(kFloor)) : h[i];
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&x);
      o[2 * i] = __uint_as_float(u << 16);
      o[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
    }
  }
};

struct Stat {
  float m, s, a;  // reference (-inf: nothing yet), sum, sum weighted with y
};
// y of x at reference M; -200 for what is too small to count (2^-200 is 0 in
// F32), which keeps 0 * inf out of the weighted sum; a NaN stays.
__device__ __forceinline__ float y_of(float x, float M) {
  const float y = near(M) ? fmaf(x, kLog2e, -(M * kLog2e)) : (x - M) * kLog2e;
  return max_nan(y, -200.f);
}
// How far sums move from reference `from` up to reference `to`, in log2 units:
// between near ones the difference of the rounded c that their y are relative to
// (a contracted product would leave one unrounded: 6e-5 off about 3000).
__device__ __forceinline__ float shift(float from, float to) {
  const float c0 = __fmul_rn(from, kLog2e), c1 = __fmul_rn(to, kLog2e);
  if (near(from)) return near(to) ? __fsub_rn(c0, c1) : -fmaf(to, kLog2e, -c0);
  return near(to) ? fmaf(from, kLog2e, -c1) : (from - to) * kLog2e;
}

// The states of a warp's lanes joined, in every lane.
__device__ __forceinline__ Stat warp_join(Stat t) {
  const float M = key_value(__reduce_max_sync(0xffffffffu, order_key(t.m)));
  if (t.m != M) {
    const float d = t.m == -INFINITY ? -INFINITY : shift(t.m, M), c = ex2f(d);
    t.a = c == 0.f ? 0.f * t.s : (t.a + t.s * d) * c;
    t.s *= c;  // a NaN carried by an empty lane stays
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
    t.a += __shfl_xor_sync(0xffffffffu, t.a, o);
  }
  return {M, t.s, t.a};
}

using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack(float a, float b) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpack(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

// A thread's running state; s and a as two partial sums each.
struct Acc {
  float m = -INFINITY;
  f32x2 s = 0, a = 0;
  __device__ __forceinline__ Stat stat() const {
    float s0, s1, a0, a1;
    unpack(s, s0, s1);
    unpack(a, a0, a1);
    return {m, s0 + s1, a0 + a1};
  }
};

__device__ __forceinline__ void move_up(Acc& st, float hi) {
  const float d = st.m == -INFINITY ? -INFINITY : shift(st.m, hi), c = ex2f(d);
  const f32x2 c2 = pack(c, c);
  // c = 0: nothing of the sums is left but a NaN where a NaN or infinity came before
  if (c != 0.f) st.a = fma2(st.s, pack(d, d), st.a);
  st.s = fma2(st.s, c2, 0);
  st.a = c != 0.f ? fma2(st.a, c2, 0) : st.s;
  st.m = hi;
}
// Terms of any values at any reference.
template <int N>
__device__ __forceinline__ void add_any(const float (&x)[N], Acc& st) {
  const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float y0 = y_of(x[i], ref), y1 = y_of(x[i + 1], ref);
    const f32x2 e = pack(ex2f(y0), ex2f(y1));
    st.s = add2(st.s, e);
    st.a = fma2(e, pack(y0, y1), st.a);
  }
}

// The row as 16-byte vectors from the aligned address at or before its
// first element: vector v holds elements v * N - lead .. + N - 1.  A vector
// that is not wholly inside the row is read element by element, -inf outside.
template <typename T>
struct Row {
  const T* x;
  int vocab, lead, nvec;
  __device__ __forceinline__ Row(const T* row, int V) : x(row), vocab(V) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    nvec = (V + lead + Elem<T>::N - 1) / Elem<T>::N;
  }
  __device__ __forceinline__ bool whole(int v) const {
    const int e = v * Elem<T>::N - lead;
    return e >= 0 && e + Elem<T>::N <= vocab;
  }
  __device__ __forceinline__ uint4 raw(int v) const {
    return __ldg(reinterpret_cast<const uint4*>(x + (long long)v * Elem<T>::N - lead));
  }
  __device__ __forceinline__ void edge(int v, float (&o)[Elem<T>::N]) const {
#pragma unroll
    for (int i = 0; i < Elem<T>::N; i++) {
      const int e = v * Elem<T>::N - lead + i;
      o[i] = e >= 0 && e < vocab ? Elem<T>::one(x[e]) : -INFINITY;
    }
  }
  __device__ __forceinline__ void load(int v, float (&o)[Elem<T>::N]) const {
    if (whole(v))
      Elem<T>::template unpack<false>(raw(v), o);
    else
      edge(v, o);
  }
  // Adds a vector at the row's ends; the maximum of what was added.
  __device__ __forceinline__ float add_edge(int v, Acc& st) const {
    float x[Elem<T>::N], hi = -INFINITY;
    edge(v, x);
#pragma unroll
    for (int i = 0; i < Elem<T>::N; i++) hi = fmaxf(hi, x[i]);
    if (hi > st.m + kSlack) move_up(st, hi);
    add_any(x, st);
    return hi;
  }
  template <int NV>
  __device__ __forceinline__ float add(const uint4 (&w)[NV], Acc& st) const {
    constexpr int N = Elem<T>::N;
    const float hi = Elem<T>::top(w);
    if (hi > st.m + kSlack) move_up(st, hi);  // also the first value above -inf
    if (near(st.m)) {
      const float c = st.m * kLog2e;
      const f32x2 l2 = pack(kLog2e, kLog2e), nc = pack(-c, -c);
#pragma unroll
      for (int q = 0; q < NV; q++) {
        float x[N];
        Elem<T>::template unpack<true>(w[q], x);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const f32x2 y = fma2(pack(x[i], x[i + 1]), l2, nc);
          float y0, y1;
          unpack(y, y0, y1);
          const f32x2 e = pack(ex2f(y0), ex2f(y1));
          st.s = add2(st.s, e);
          st.a = fma2(e, y, st.a);
        }
      }
    } else {  // nothing seen yet but -inf, or a far reference
#pragma unroll
      for (int q = 0; q < NV; q++) {
        float x[N];
        Elem<T>::template unpack<false>(w[q], x);
        add_any(x, st);
      }
    }
    return hi;
  }
};

__device__ __forceinline__ float logprob_of(float x, float M, float ln_s) {
  // as y_of, but a far smaller logit keeps its distance
  const float d = near(M) && x > kFloor ? fmaf(x, kLog2e, -(M * kLog2e)) * kLn2 : x - M;
  return d - ln_s;
}

struct LpShared {
  uint32_t seg[kMaxSeg];  // order keys of the segments' maxima (the leader's: all of the row)
  Stat warp[32];
  Stat cta[8];            // the leader's: one per CTA of the cluster
  int sel[LAYA_MAX_TOP];
  uint32_t t;
  int n_cand;
  int wcount[33];
  unsigned long long best;
  uint64_t full[kMaxStages], empty[kMaxStages];
};
// Dynamic shared memory: the ring, and after the pass the list of the best
// elements (order keys, then indices).
extern __shared__ __align__(128) uint4 lp_dyn[];

// The kk best of nseg <= 32 Q segments, by one warp: the best of all, kk times
// (a rank of each segment among all took six times the instructions, which
// the rows that are still being read miss: 2048 rows of 152064, 5
// alternatives, 129 us against 125).  The last one's key.
template <int Q>
__device__ __forceinline__ uint32_t best_segments(LpShared& sh, int nseg, int kk) {
  const int lane = threadIdx.x % 32;
  uint32_t k[Q], best = 0;
#pragma unroll
  for (int q = 0; q < Q; q++) k[q] = q * 32 + lane < nseg ? sh.seg[q * 32 + lane] : 0;
#pragma unroll 1
  for (int n = 0; n < kk; n++) {
    best = 0;
#pragma unroll
    for (int q = 0; q < Q; q++) best = max(best, k[q]);
    best = __reduce_max_sync(0xffffffffu, best);
    int first = kMaxSeg;
#pragma unroll
    for (int q = Q - 1; q >= 0; q--)
      if (k[q] == best) first = q * 32 + lane;
    first = __reduce_min_sync(0xffffffffu, first);
#pragma unroll
    for (int q = 0; q < Q; q++)
      if (q * 32 + lane == first) k[q] = 0;  // below every key
    if (lane == 0) sh.sel[n] = first;
  }
  return best;
}

// The `top` best elements of the row, by the leader CTA, all threads.  Run once
// per row, so written for few instructions rather than few cycles: unrolled, it
// cost more in instruction fetches than in work.  2048 rows of 152064 in BF16
// take 125 us with 5 alternatives and 101 without.  Rows whose large values lie
// together are slow: sorted ones 193 us with 5 alternatives, 6.7 ms with 64
// (against 128 and 211 for random ones, same run).
template <typename T>
__device__ void pick_top(const LpArgs& p, const Row<T>& row, int nseg, LpShared& sh, float M, float ln_s,
                         long long r) {
  constexpr int N = Elem<T>::N;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid % 32, warp = tid / 32, seg_vec = p.seg_vec;
  uint32_t* ckey = reinterpret_cast<uint32_t*>(lp_dyn);
  int* cidx = reinterpret_cast<int*>(ckey + kCand);
  const int kk = min(p.top, nseg);
  if (warp == 0) {
    const uint32_t last = nseg <= 256 ? best_segments<8>(sh, nseg, kk) : best_segments<kMaxSeg / 32>(sh, nseg, kk);
    // the last chosen segment's maximum; fewer segments than `top`: everything counts
    if (lane == 0) sh.t = nseg < p.top ? kNegInfKey : max(last, kNegInfKey);
  }
  if (tid == 0) sh.n_cand = 0;
  __syncthreads();
  const uint32_t t = sh.t;
  const float tv = key_value(t);
  const int nv = kk * seg_vec, log_sv = __ffs(seg_vec) - 1;
  auto vec_of = [&](int i) { return (sh.sel[i >> log_sv] << log_sv) + (i & (seg_vec - 1)); };
  // List the chosen segments' elements from t on; if those are too many (many
  // equal to t), the ones beyond t.
  bool above = t == kNegInfKey;
  int have;
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i0 = tid; i0 < nv; i0 += 4 * nt) {
      uint4 w[4];
      uint32_t look = 0;  // which of the four may hold some
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int v = i0 + q * nt < nv ? vec_of(i0 + q * nt) : row.nvec;
        if (row.whole(v)) {
          w[q] = row.raw(v);
          look |= 1u << q;
        } else if (v < row.nvec) {
          look |= 16u << q;  // at the row's ends
        }
      }
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint4 x[1] = {w[q]};
        if ((look >> q & 1) && !(Elem<T>::top(x) >= tv)) look &= ~(1u << q);
      }
#pragma unroll 1
      for (; look; look &= look - 1) {
        const int bit = __ffs(look) - 1, q = bit & 3, v = vec_of(i0 + q * nt), first = v * N - row.lead;
        float x[N];
        if (bit < 4) {
          uint4 u = w[0];
          if (q == 1) u = w[1];
          if (q == 2) u = w[2];
          if (q == 3) u = w[3];
          Elem<T>::template unpack<false>(u, x);
        } else {
          row.edge(v, x);
        }
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < N; e++) hits |= ((above ? x[e] > tv : x[e] >= tv) ? 1u : 0u) << e;
#pragma unroll 1
        for (; hits; hits &= hits - 1) {
          const int e = first + __ffs(hits) - 1, at = atomicAdd(&sh.n_cand, 1);
          if (at < kCand) {
            ckey[at] = order_key(Elem<T>::one(row.x[e]));
            cidx[at] = e;
          }
        }
      }
    }
    __syncthreads();
    have = sh.n_cand;
    if (have <= kCand || above) break;
    above = true;
    __syncthreads();
    if (tid == 0) sh.n_cand = 0;
    __syncthreads();
  }
  int* ids = p.ids + r * p.top;
  float* tlp = p.tlp + r * p.top;
  if (have > kCand) {
    // More elements above t than the list holds (a row whose large values
    // lie together): the best after the last one found, `top` times.
    unsigned long long last = ~0ull;
#pragma unroll 1
    for (int n = 0; n < p.top; n++) {
      if (tid == 0) sh.best = 0;
      __syncthreads();
      unsigned long long b = 0;
#pragma unroll 1
      for (int i = tid; i < nv; i += nt) {
        const int v = vec_of(i);
        if (v >= row.nvec) continue;
        float x[N];
        row.load(v, x);
#pragma unroll
        for (int e = 0; e < N; e++) {
          const unsigned long long k =
              ((unsigned long long)order_key(x[e]) << 32) | (0xffffffffu - (uint32_t)(v * N - row.lead + e));
          if (k < last && k > b) b = k;
        }
      }
      atomicMax(&sh.best, b);
      __syncthreads();
      last = sh.best;
      if (tid == 0) {
        ids[n] = (int)(0xffffffffu - (uint32_t)last);
        tlp[n] = logprob_of(key_value((uint32_t)(last >> 32)), M, ln_s);
      }
      __syncthreads();
    }
    return;
  }
  if (above && t > kNegInfKey && have < p.top) {
    // the first elements equal to t, in index order: the chosen segments by
    // index, a vector per thread at a time
    if (warp == 0) {
      int mine[2], rank[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int i = lane + 32 * h;
        mine[h] = i < kk ? sh.sel[i] : 0x7fffffff;
        rank[h] = 0;
#pragma unroll 1
        for (int j = 0; j < kk; j++) rank[h] += sh.sel[j] < mine[h];
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; h++)
        if (lane + 32 * h < kk) sh.sel[rank[h]] = mine[h];
    }
    __syncthreads();
    const int need = p.top - have;
    int found = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < nv && found < need; i0 += nt) {
      const int i = i0 + tid;
      uint32_t mask = 0;
      int v = 0;
      if (i < nv) {
        v = vec_of(i);
        if (v < row.nvec) {
          float x[N];
          row.load(v, x);
#pragma unroll
          for (int e = 0; e < N; e++) mask |= (order_key(x[e]) == t ? 1u : 0u) << e;
        }
      }
      const int c = __popc(mask);
      int inc = c;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) sh.wcount[warp] = inc;
      __syncthreads();
      int before = found + inc - c, all = found;
#pragma unroll 1
      for (int w = 0; w < nt / 32; w++) {
        if (w < warp) before += sh.wcount[w];
        all += sh.wcount[w];
      }
#pragma unroll 1
      for (uint32_t left = mask; left && before < need; left &= left - 1, before++) {
        ckey[have + before] = t;
        cidx[have + before] = v * N - row.lead + __ffs(left) - 1;
      }
      found = all;
      __syncthreads();
    }
    have += min(found, need);
  }
#pragma unroll 1
  for (int i = tid; i < max(have, p.top); i += nt) {
    if (i >= have) {
      ids[i] = -1;
      tlp[i] = -INFINITY;
      continue;
    }
    const uint32_t ki = ckey[i];
    const int xi = cidx[i];
    int rank = 0;
#pragma unroll 1
    for (int j = 0; j < have; j++) rank += ckey[j] > ki || (ckey[j] == ki && cidx[j] < xi);
    if (rank < p.top) {
      ids[rank] = xi;
      tlp[rank] = logprob_of(key_value(ki), M, ln_s);
    }
  }
}

// One row per cluster of C CTAs (1, 2, 4 or 8); the leader (rank 0) receives
// every CTA's state and segment maxima through distributed shared memory and
// finishes the row.
//   RING  : long rows.  CTA c takes chunks c, c + C, ... of 1024 vectors; a
//           producer warp brings them with 1-D bulk copies into a ring, so that
//           the bytes in flight do not sit in registers, and each of the eight
//           consumer warps takes 128 vectors of a chunk.
//   else  : short rows, 32 vectors per warp at a time into registers.
template <typename T, bool TOP, bool RING>
__global__ void __launch_bounds__(RING ? 32 * (kRingWarps + 1) : 256, 4)
    token_logprobs_kernel(const LpArgs p, int C) {
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, nw = blockDim.x / 32;
  const long long r = blockIdx.x / C;
  const int rank = blockIdx.x % C;
  const Row<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  const int qrows = (row.nvec + 31) / 32;  // rows of 32 vectors
  const int nseg = (row.nvec + p.seg_vec - 1) / p.seg_vec;
  const int lo = row.lead ? 1 : 0, hi = (int)(((long long)p.vocab + row.lead) / Elem<T>::N);  // whole vectors
  const int chunks = (row.nvec + kChunk - 1) / kChunk;
  auto copy_chunk = [&](int c, int st) {
    const int a = max(c * kChunk, lo), b = min((c + 1) * kChunk, hi);
    if (b > a) {
      mbar_expect_tx(&sh.full[st], (uint32_t)(b - a) * 16);
      bulk_g2s(lp_dyn + st * kChunk + (a - c * kChunk), row.x + (long long)a * Elem<T>::N - row.lead,
               (uint32_t)(b - a) * 16, &sh.full[st]);
    } else {
      mbar_arrive(&sh.full[st]);
    }
  };
  if (RING && tid == 32 * kRingWarps) {  // the producer: the first stages at once
    for (int i = 0; i < p.stages; i++) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], kRingWarps);
    }
    mbar_fence_init();
    for (int i = 0, c = rank; i < p.stages && c < chunks; i++, c += C) copy_chunk(c, i);
  }
  if (TOP && rank == 0)
    for (int i = tid; i < nseg; i += blockDim.x) sh.seg[i] = 0;
  // the given tokens' logits, early: their latency hides behind the pass
  float xt = 0.f;
  int tok = -1;
  if (rank == 0 && tid < p.n_tok) tok = p.tokens[r * p.tstride + tid];
  auto put_seg = [&](int s, uint32_t key) {
    if (C == 1)
      atomicMax(&sh.seg[s], key);
    else
      asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(cluster_addr(&sh.seg[s], 0)), "r"(key)
                   : "memory");
  };
  if (C > 1)
    cluster_sync();  // the leader's shared memory is ready
  else
    __syncthreads();
  if (tok >= 0 && tok < p.vocab) xt = Elem<T>::one(row.x[tok]);
  Acc acc;
  if constexpr (RING) {
    bool live = true;
    if (warp == kRingWarps) {
      if (lane == 0) {
        int n = min(p.stages, chunks > rank ? (chunks - rank + C - 1) / C : 0);  // chunks asked for
        for (int c = rank + n * C; c < chunks && live; c += C) {
          const int st = n % p.stages;
          live = mbar_wait(&sh.empty[st], ((n / p.stages) & 1) ^ 1, kBudget);
          if (live) {
            copy_chunk(c, st);
            n++;
          }
        }
        // no copy is in flight when the CTA ends or the ring is reused
        for (int i = max(0, n - p.stages); i < n; i++)
          live = mbar_wait(&sh.full[i % p.stages], (i / p.stages) & 1, kBudget) && live;
      }
    } else {
      for (int c = rank, i = 0; c < chunks; c += C, i++) {
        const int st = i % p.stages, v0 = c * kChunk + warp * 128;
        live = __all_sync(0xffffffffu, mbar_wait(&sh.full[st], (i / p.stages) & 1, kBudget));
        if (!live) break;
        const uint4* src = lp_dyn + st * kChunk + warp * 128 + lane;
        float smax = -INFINITY;
        if (v0 >= lo && v0 + 128 <= hi) {
          const uint4 w[4] = {src[0], src[32], src[64], src[96]};
          smax = row.add(w, acc);
        } else {
#pragma unroll 1
          for (int q = 0; q < 4; q++) {
            const int v = v0 + q * 32 + lane;
            if (v >= lo && v < hi) {
              const uint4 w[1] = {src[q * 32]};
              smax = fmaxf(smax, row.add(w, acc));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[st]);
        if (TOP && v0 < row.nvec) {  // a segment is a multiple of 128 vectors
          const uint32_t key = __reduce_max_sync(0xffffffffu, order_key(smax));
          if (lane == 0) put_seg(v0 / p.seg_vec, key);
        }
      }
      // the row's first and last vector, where they are not whole
      if (rank == 0 && warp == 0 && lane < 2) {
        const int v = lane ? max(hi, lo) : 0;
        if (lane ? v < row.nvec : lo == 1) {
          const float m = row.add_edge(v, acc);
          if (TOP) put_seg(v / p.seg_vec, order_key(m));
        }
      }
    }
    if (!live && lane == 0) atomicOr(p.status, LAYA_STATUS_TIMEOUT);
  } else {
    // a segment is the vectors of seg_vec <= 32 neighbouring lanes
    for (int q = rank * nw + warp; q < qrows; q += C * nw * 4) {
      uint4 w[4];
      float m[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int v = (q + e * C * nw) * 32 + lane;
        if (row.whole(v)) w[e] = row.raw(v);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int v = (q + e * C * nw) * 32 + lane;
        const uint4 x[1] = {w[e]};
        m[e] = row.whole(v) ? row.add(x, acc) : v < row.nvec ? row.add_edge(v, acc) : -INFINITY;
      }
      if (TOP) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          for (int o = 1; o < p.seg_vec; o <<= 1) m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], o));
          const int v = (q + e * C * nw) * 32 + lane;
          if (lane % p.seg_vec == 0 && v < row.nvec) put_seg(v / p.seg_vec, order_key(m[e]));
        }
      }
    }
  }
  Stat st = warp_join(acc.stat());
  if (lane == 0) sh.warp[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st = warp_join(lane < nw ? sh.warp[lane] : Stat{-INFINITY, 0.f, 0.f});
    if (lane == 0) {
      if (C == 1) {
        sh.cta[0] = st;
      } else {
        const uint32_t a = cluster_addr(&sh.cta[rank], 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(st.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a + 4), "f"(st.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a + 8), "f"(st.a) : "memory");
      }
    }
  }
  if (C > 1) {
    cluster_sync();
    if (rank) return;
    st = warp_join(lane < C ? sh.cta[lane] : Stat{-INFINITY, 0.f, 0.f});
  } else {
    __syncthreads();
    st = sh.cta[0];
  }
  const bool none = st.m == -INFINITY && st.s == 0.f;  // every logit -inf
  const bool bad = !none && !(st.s > 0.f && st.s < INFINITY && st.m < INFINITY);
  const float M = bad ? NAN : st.m;
  const float ln_s = none ? 0.f : logf(st.s);
  if (tid == 0) {
    // a near reference is c ln 2: M, and what rounding M log2 e left out
    const float rest = near(M) ? fmaf(-M, kLog2e, M * kLog2e) * kLn2 : 0.f;
    if (p.lse) p.lse[r] = none ? -INFINITY : bad ? NAN : M + (ln_s + rest);
    if (p.ent) p.ent[r] = none ? 0.f : bad ? NAN : ln_s - kLn2 * (st.a / st.s);
  }
  for (int j = tid; j < p.n_tok; j += blockDim.x) {
    if (j >= (int)blockDim.x) {
      tok = p.tokens[r * p.tstride + j];
      if (tok >= 0 && tok < p.vocab) xt = Elem<T>::one(row.x[tok]);
    }
    const bool in = tok >= 0 && tok < p.vocab;
    if (!in && tok != -1) atomicOr(p.status, LAYA_STATUS_TOKEN);
    p.lp[r * p.n_tok + j] = !in ? 0.f : none ? -INFINITY : bad ? NAN : logprob_of(xt, M, ln_s);
  }
  if (TOP) {
    if (none || bad) {
      for (int i = tid; i < p.top; i += blockDim.x) {
        p.ids[r * p.top + i] = -1;
        p.tlp[r * p.top + i] = bad ? NAN : -INFINITY;
      }
    } else {
      pick_top<T>(p, row, nseg, sh, M, ln_s, r);
    }
  }
}

template <typename T, bool TOP, bool RING>
int launch_logprobs(const LpArgs& p, int C, int threads, const DeviceInfo& di, cudaStream_t st) {
  constexpr int kMaxDyn = kMaxStages * kChunk * 16;
  static std::atomic<bool> configured[64];
  if (!configured[di.device & 63]) {
    LAYA_CK(cudaFuncSetAttribute(token_logprobs_kernel<T, TOP, RING>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kMaxDyn));
    configured[di.device & 63] = true;
  }
  const long long grid = (long long)p.rows * C;
  if (grid > 0x7fffffffll) return fail(LAYA_E_INVALID, "too many logit rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = std::max(RING ? p.stages * kChunk * 16 : 0, TOP ? kCand * 8 : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  LAYA_CK(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, TOP, RING>, (const LpArgs)p, C));
  return 0;
}

template <typename T>
int logprobs_go(LpArgs p, const DeviceInfo& di, cudaStream_t st) {
  const int N = Elem<T>::N;
  // Segments: the more, the less is read again for the `top` (top / segments
  // of the row), the fewer, the cheaper their choice: eight per alternative, 256
  // at least; always more than LAYA_MAX_TOP, or one per vector.
  const long long nvec = ((long long)p.vocab + 2 * N - 2) / N;  // with any misalignment
  const long long most = std::min(kMaxSeg, std::max(256, p.top * 8));
  p.seg_vec = 1;
  while (nvec > p.seg_vec * most) p.seg_vec *= 2;
  // The ring form keeps one maximum per 128 vectors: rows that still give
  // twice `top` segments, 24 at least.
  const bool ring = nvec >= 128ll * std::max(24, 2 * p.top);
  if (ring) p.seg_vec = std::max(p.seg_vec, 128);
  // Few rows: a cluster of CTAs per row, as long as a CTA keeps a chunk of it
  // (8 KB of a short one) and the CTAs fit the GPU at once.
  int C = 1;
  while (C < 8 && (long long)p.rows * C * 2 <= 2 * di.sms && nvec / (2 * C) >= (ring ? kChunk : kChunk / 2)) C *= 2;
  if (ring) {
    // four CTAs per SM with three stages each, or few with deep rings
    const long long chunks = (nvec + kChunk - 1) / kChunk;
    const bool few = (long long)p.rows * C <= 2 * di.sms;
    p.stages = (int)std::min<long long>(few ? 6 : 3, (chunks + C - 1) / C);
    const int threads = 32 * (kRingWarps + 1);
    return p.top ? launch_logprobs<T, true, true>(p, C, threads, di, st)
                 : launch_logprobs<T, false, true>(p, C, threads, di, st);
  }
  const int threads = nvec <= kChunk ? 128 : 256;
  return p.top ? launch_logprobs<T, true, false>(p, C, threads, di, st)
               : launch_logprobs<T, false, false>(p, C, threads, di, st);
}

}  // namespace

int token_logprobs(uint32_t type, const void* logits, int64_t row_stride, int rows, int vocab, const int32_t* tokens,
                   int64_t token_stride, int n_tokens, int top, float* logprobs, float* entropy, float* lse,
                   int32_t* top_ids, float* top_logprobs, unsigned* status, cudaStream_t st) {
  if (type != LAYA_TYPE_F32 && type != LAYA_TYPE_F16 && type != LAYA_TYPE_BF16)
    return fail(LAYA_E_INVALID, "logits must be F32, F16 or BF16");
  if (rows < 0 || vocab < 1 || n_tokens < 0) return fail(LAYA_E_INVALID, "invalid logits size");
  if (vocab > (1 << 30)) return fail(LAYA_E_INVALID, "vocabulary too large");
  if (top < 0 || top > LAYA_MAX_TOP) return fail(LAYA_E_INVALID, "top must be 0..64");
  if (row_stride < 0 || token_stride < 0) return fail(LAYA_E_INVALID, "negative row stride");
  if (rows == 0) return 0;
  if (!logits || (n_tokens && (!tokens || !logprobs)) || (top && (!top_ids || !top_logprobs)))
    return fail(LAYA_E_INVALID, "null argument");
  if (reinterpret_cast<uintptr_t>(logits) % (type == LAYA_TYPE_F32 ? 4 : 2))
    return fail(LAYA_E_INVALID, "misaligned logits");
  DeviceInfo di;
  if (int rc = device_info(&di)) return rc;
  LpArgs p{logits,   row_stride, rows, vocab,   tokens,       token_stride, n_tokens,
           top,      logprobs,   entropy, lse,  top_ids,      top_logprobs, status ? status : di.status, 1, 0};
  if (type == LAYA_TYPE_F32) return logprobs_go<float>(p, di, st);
  if (type == LAYA_TYPE_F16) return logprobs_go<half>(p, di, st);
  return logprobs_go<__nv_bfloat16>(p, di, st);
}

}  // namespace laya

using namespace laya;

extern "C" int laya_token_logprobs(uint32_t type, const void* logits, int64_t row_stride, int rows, int vocab,
                                   const int32_t* tokens, int64_t token_stride, int n_tokens, int top,
                                   float* logprobs, float* entropy, float* lse, int32_t* top_ids, float* top_logprobs,
                                   void* stream) {
  return guarded([&]() -> int {
    return token_logprobs(type, logits, row_stride, rows, vocab, tokens, token_stride, n_tokens, top, logprobs, entropy,
                          lse, top_ids, top_logprobs, nullptr, static_cast<cudaStream_t>(stream));
  });
}
