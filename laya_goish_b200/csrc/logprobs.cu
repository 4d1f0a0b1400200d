// Log probabilities of given tokens, entropy and the likeliest tokens of
// full-vocabulary logit rows, each row read once.
//
// With any reference M near the row's maximum,
//   s = sum e^(x - M),  a = sum e^(x - M) (x - M),
//   lse = M + ln s,  logprob_j = (x_j - M) - ln s,  entropy = ln s - a / s.
// Every thread keeps its own (M, s, a) and moves M only when a value passes
// it by more than 4 (e^4 per term costs no precision in F32), so the rescale
// is rare; the threads' states are merged at the end.
//
// The `top` best come from the same pass: the row is cut into contiguous
// segments and the pass leaves each segment's maximum in shared memory.
// Order elements by (value descending, index ascending) and segments by
// (maximum descending, index ascending): an element outside the best `top`
// segments is preceded by the maxima of `top` segments, so the best `top`
// elements lie in the best `top` segments, ties included, whatever the row
// holds.  Only those segments are read again (from L2): elements above the
// last chosen segment's maximum t go to a list, and if there are fewer than
// `top` of them the first elements equal to t follow in index order.
//
// Bound by HBM (the row's bytes) with the exponentials close behind: one per
// element, 16 per SM and clock.
#include <algorithm>

#include "device_ops.h"
#include "launch.h"
#include "ptx.cuh"

namespace laya {

namespace {

constexpr int kMaxSeg = 256;   // segments per row
constexpr int kCand = 1024;    // list of elements above t

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
  int seg_rows;  // > 0: 32-vector rows per segment; < 0: a segment is -seg_rows lanes' vectors
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
// u32 of the same order; -0 counts as +0
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kNegInfKey = 0x007fffffu;  // order_key(-inf)

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[4]) {
    o[0] = __uint_as_float(v.x);
    o[1] = __uint_as_float(v.y);
    o[2] = __uint_as_float(v.z);
    o[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(float x) { return x; }
};
template <>
struct Elem<half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const half2*>(&w[i]));
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(half x) { return __half2float(x); }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
};

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
      Elem<T>::unpack(raw(v), o);
    else
      edge(v, o);
  }
};

struct Stat {
  float m, s, a;  // reference (-inf: nothing yet), sum, weighted sum
};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 4.f;

// b's sums moved to a's reference or the other way round, then added.
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float M = fmaxf(a.m, b.m);
  if (M == -INFINITY) return {M, a.s + b.s, a.a + b.a};  // empty, or NaN carried in s
  Stat r{M, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const Stat& t = i ? b : a;
    if (t.m == -INFINITY) {
      r.s += t.s;
      r.a += t.a;
    } else {
      const float d = t.m - M, c = ex2f(d * kLog2e);  // d: 0, or a move down
      r.s += t.s * c;
      r.a += c == 0.f ? 0.f * t.s : (t.a + t.s * d) * c;
    }
  }
  return r;
}

template <int N>
__device__ __forceinline__ void accumulate(const float (&x)[N], float vmax, Stat& st) {
  if (vmax > st.m + kSlack) {  // also the first value above -inf
    const float d = st.m - vmax, c = ex2f(d * kLog2e);
    if (c == 0.f) {
      st.s *= 0.f;  // 0, or NaN where a NaN or infinity came before
      st.a = st.s;
    } else {
      st.a = (st.a + st.s * d) * c;
      st.s *= c;
    }
    st.m = vmax;
  }
  const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int i = 0; i < N; i++) {
    // below -150 the term is 0 in F32; the bound keeps 0 * -inf out of a
    const float d = max_nan(x[i] - ref, -150.f);
    const float e = ex2f(d * kLog2e);
    st.s += e;
    st.a = fmaf(e, d, st.a);
  }
}

template <int N>
__device__ __forceinline__ float vec_max(const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; i++) m = fmaxf(m, x[i]);
  return m;
}

struct LpShared {
  uint32_t seg[kMaxSeg];  // order keys of the segments' maxima (the leader's: all of the row)
  Stat warp[32];
  Stat cta[16];           // the leader's: one per CTA of the cluster
  int sel[LAYA_MAX_TOP];
  uint32_t ckey[kCand];
  int cidx[kCand];
  int n_cand, n_tie;
  int wcount[33];
  unsigned long long best;
};

// The `top` best elements of the row, by the leader CTA, all threads.
template <typename T>
__device__ void pick_top(const LpArgs& p, const Row<T>& row, int nseg, int seg_vec, LpShared& sh, float M, float ln_s,
                         long long r) {
  constexpr int N = Elem<T>::N;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid % 32, warp = tid / 32;
  const int kk = min(p.top, nseg);
  if (tid == 0) sh.n_cand = sh.n_tie = 0;
  // rank of each segment among all
  for (int i = tid; i < nseg; i += nt) {
    const uint32_t ki = sh.seg[i];
    int rank = 0;
    for (int j = 0; j < nseg; j++) {
      const uint32_t kj = sh.seg[j];
      rank += kj > ki || (kj == ki && j < i);
    }
    if (rank < kk) sh.sel[rank] = i;
  }
  __syncthreads();
  // the last chosen segment's maximum; fewer segments than `top`: everything counts
  const uint32_t t = nseg < p.top ? kNegInfKey : max(sh.seg[sh.sel[kk - 1]], kNegInfKey);
  const int nv = kk * seg_vec;
  for (int i = tid; i < nv; i += nt) {
    const int v = sh.sel[i / seg_vec] * seg_vec + i % seg_vec;
    if (v >= row.nvec) continue;
    float x[N];
    row.load(v, x);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const uint32_t k = order_key(x[e]);
      if (k > t) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) {
          sh.ckey[at] = k;
          sh.cidx[at] = v * N - row.lead + e;
        }
      }
    }
  }
  __syncthreads();
  int have = sh.n_cand;
  int* ids = p.ids + r * p.top;
  float* tlp = p.tlp + r * p.top;
  if (have > kCand) {
    // More elements above t than the list holds (a row whose large values
    // lie together): the best after the last one found, `top` times.
    unsigned long long last = ~0ull;
    for (int n = 0; n < p.top; n++) {
      if (tid == 0) sh.best = 0;
      __syncthreads();
      unsigned long long b = 0;
      for (int i = tid; i < nv; i += nt) {
        const int v = sh.sel[i / seg_vec] * seg_vec + i % seg_vec;
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
        tlp[n] = (key_value((uint32_t)(last >> 32)) - M) - ln_s;
      }
      __syncthreads();
    }
    return;
  }
  if (have < p.top && t > kNegInfKey) {
    // the first elements equal to t, in index order: the chosen segments by
    // index, a vector per thread at a time
    if (tid < 32) {
      int mine[2], rank[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int i = tid + 32 * h;
        mine[h] = i < kk ? sh.sel[i] : 0x7fffffff;
        rank[h] = 0;
        for (int j = 0; j < kk; j++) rank[h] += sh.sel[j] < mine[h];
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; h++)
        if (tid + 32 * h < kk) sh.sel[rank[h]] = mine[h];
    }
    __syncthreads();
    const int need = p.top - have;
    int found = 0;
    for (int i0 = 0; i0 < nv && found < need; i0 += nt) {
      const int i = i0 + tid;
      uint32_t mask = 0;
      int v = 0;
      if (i < nv) {
        v = sh.sel[i / seg_vec] * seg_vec + i % seg_vec;
        if (v < row.nvec) {
          float x[N];
          row.load(v, x);
#pragma unroll
          for (int e = 0; e < N; e++) mask |= (order_key(x[e]) == t ? 1u : 0u) << e;
        }
      }
      const int c = __popc(mask);
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) sh.wcount[warp] = inc;
      __syncthreads();
      int before = found + inc - c, all = found;
      for (int w = 0; w < nt / 32; w++) {
        if (w < warp) before += sh.wcount[w];
        all += sh.wcount[w];
      }
      for (uint32_t left = mask; left && before < need; left &= left - 1, before++) {
        sh.ckey[have + before] = t;
        sh.cidx[have + before] = v * N - row.lead + __ffs(left) - 1;
      }
      found = all;
      __syncthreads();
    }
    have += min(found, need);
  }
  for (int i = tid; i < p.top; i += nt)
    if (i >= have) {
      ids[i] = -1;
      tlp[i] = -INFINITY;
    }
  for (int i = tid; i < have; i += nt) {
    const uint32_t ki = sh.ckey[i];
    const int xi = sh.cidx[i];
    int rank = 0;
    for (int j = 0; j < have; j++) rank += sh.ckey[j] > ki || (sh.ckey[j] == ki && sh.cidx[j] < xi);
    if (rank < p.top) {
      ids[rank] = xi;
      tlp[rank] = (key_value(ki) - M) - ln_s;
    }
  }
}

// One row per cluster of CTAs (cluster size 1, 2, 4 or 8): CTA c takes the
// segments or 32-vector rows c, c + C, ... through its warps; the leader
// (rank 0) receives every CTA's state and segment maxima through distributed
// shared memory and finishes the row.
template <typename T, bool TOP>
__global__ void __launch_bounds__(512) token_logprobs_kernel(const LpArgs p, int C) {
  constexpr int N = Elem<T>::N;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, nw = blockDim.x / 32;
  const long long r = blockIdx.x / C;
  const int rank = blockIdx.x % C;
  const Row<T> row(static_cast<const T*>(p.x) + r * p.stride, p.vocab);
  // the given tokens' logits, early: their latency hides behind the pass
  float xt = 0.f;
  int tok = -1;
  if (rank == 0 && tid < p.n_tok) {
    tok = p.tokens[r * p.tstride + tid];
    if (tok >= 0 && tok < p.vocab) xt = Elem<T>::one(row.x[tok]);
  }
  auto put_seg = [&](int s, uint32_t key) {
    if (C == 1) {
      sh.seg[s] = key;
    } else {
      const uint32_t a = cluster_addr(&sh.seg[s], 0);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(key) : "memory");
    }
  };
  if (C > 1) cluster_sync();  // the leader's shared memory exists
  Stat st{-INFINITY, 0.f, 0.f};
  const int qrows = (row.nvec + 31) / 32;  // rows of 32 vectors
  int nseg, seg_vec;
  if (p.seg_rows > 0) {
    // segments of seg_rows (a multiple of 4) 32-vector rows, one per warp at a time
    seg_vec = p.seg_rows * 32;
    nseg = (qrows + p.seg_rows - 1) / p.seg_rows;
    for (int s = rank * nw + warp; s < nseg; s += C * nw) {
      float smax = -INFINITY;
      for (int u = 0; u < p.seg_rows; u += 4) {
        const int v0 = (s * p.seg_rows + u) * 32 + lane;
        if (row.whole(v0) && row.whole(v0 + 96)) {
          uint4 w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = row.raw(v0 + 32 * e);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float x[N];
            Elem<T>::unpack(w[e], x);
            const float m = vec_max(x);
            accumulate(x, m, st);
            smax = fmaxf(smax, m);
          }
        } else {
#pragma unroll 1
          for (int e = 0; e < 4; e++) {
            if (v0 + 32 * e >= row.nvec) break;
            float x[N];
            row.load(v0 + 32 * e, x);
            const float m = vec_max(x);
            accumulate(x, m, st);
            smax = fmaxf(smax, m);
          }
        }
      }
      if (TOP) {
        const uint32_t k = __reduce_max_sync(0xffffffffu, order_key(smax));
        if (lane == 0) put_seg(s, k);
      }
    }
  } else {
    // short rows: a segment is the vectors of `lanes` neighbouring lanes
    const int lanes = -p.seg_rows;
    seg_vec = lanes;
    nseg = (row.nvec + lanes - 1) / lanes;
    for (int q = rank * nw + warp; q < qrows; q += C * nw * 2) {
      float x[2][N], m[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int v = (q + e * C * nw) * 32 + lane;
        if (v < row.nvec) {
          row.load(v, x[e]);
        } else {
#pragma unroll
          for (int i = 0; i < N; i++) x[e][i] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        m[e] = vec_max(x[e]);
        accumulate(x[e], m[e], st);
      }
      if (TOP) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          for (int o = 1; o < lanes; o <<= 1) m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], o));
          const int v = (q + e * C * nw) * 32 + lane;
          if (lane % lanes == 0 && v < row.nvec) put_seg(v / lanes, order_key(m[e]));
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Stat b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                 __shfl_xor_sync(0xffffffffu, st.a, o)};
    st = join(st, b);
  }
  if (lane == 0) sh.warp[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st = lane < nw ? sh.warp[lane] : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const Stat b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                   __shfl_xor_sync(0xffffffffu, st.a, o)};
      st = join(st, b);
    }
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
  } else {
    __syncthreads();
  }
  st = sh.cta[0];
  for (int c = 1; c < C; c++) st = join(st, sh.cta[c]);
  const bool none = st.m == -INFINITY && st.s == 0.f;  // every logit -inf
  const bool bad = !none && !(st.s > 0.f && st.s < INFINITY && st.m < INFINITY);
  const float M = bad ? NAN : st.m;
  const float ln_s = none ? 0.f : logf(st.s);
  if (tid == 0) {
    if (p.lse) p.lse[r] = bad ? NAN : M + ln_s;
    if (p.ent) p.ent[r] = none ? 0.f : bad ? NAN : ln_s - st.a / st.s;
  }
  for (int j = tid; j < p.n_tok; j += blockDim.x) {
    if (j >= (int)blockDim.x) {
      tok = p.tokens[r * p.tstride + j];
      if (tok >= 0 && tok < p.vocab) xt = Elem<T>::one(row.x[tok]);
    }
    const bool in = tok >= 0 && tok < p.vocab;
    if (!in && tok != -1) atomicOr(p.status, LAYA_STATUS_TOKEN);
    p.lp[r * p.n_tok + j] = !in ? 0.f : none ? -INFINITY : bad ? NAN : (xt - M) - ln_s;
  }
  if (TOP) {
    if (none || bad) {
      for (int i = tid; i < p.top; i += blockDim.x) {
        p.ids[r * p.top + i] = -1;
        p.tlp[r * p.top + i] = bad ? NAN : -INFINITY;
      }
    } else {
      pick_top<T>(p, row, nseg, seg_vec, sh, M, ln_s, r);
    }
  }
}

template <typename T>
int logprobs_go(LpArgs p, int sms, cudaStream_t st) {
  const int N = Elem<T>::N;
  // Segments: at most kMaxSeg per row.  Long rows take whole 32-vector rows
  // (a multiple of the four loads a warp keeps in flight); shorter ones the
  // vectors of 1..32 neighbouring lanes, so that even a few thousand entries
  // give more than LAYA_MAX_TOP segments.
  const long long nvec = ((long long)p.vocab + 2 * N - 2) / N;  // with any misalignment
  if (nvec > 32 * kMaxSeg) {
    p.seg_rows = (int)((nvec + 32ll * 4 * kMaxSeg - 1) / (32ll * 4 * kMaxSeg)) * 4;
  } else {
    int lanes = 1;
    while (nvec > (long long)lanes * kMaxSeg) lanes *= 2;
    p.seg_rows = -lanes;
  }
  // Few rows: a cluster of CTAs per row, as long as a CTA keeps 8 KB of it
  // and the CTAs fit the GPU at once.
  int C = 1;
  while (C < 8 && (long long)p.rows * C * 2 <= 2 * sms && (long long)p.vocab * (int)sizeof(T) / (2 * C) >= 8192) C *= 2;
  const int threads = 256;
  const long long grid = (long long)p.rows * C;
  if (grid > 0x7fffffffll) return fail(LAYA_E_INVALID, "too many logit rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  LAYA_CK(p.top ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, (const LpArgs)p, C)
                : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, (const LpArgs)p, C));
  return 0;
}

}  // namespace

}  // namespace laya

using namespace laya;

extern "C" int laya_token_logprobs(uint32_t type, const void* logits, int64_t row_stride, int rows, int vocab,
                                   const int32_t* tokens, int64_t token_stride, int n_tokens, int top,
                                   float* logprobs, float* entropy, float* lse, int32_t* top_ids, float* top_logprobs,
                                   void* stream) {
  return guarded([&]() -> int {
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
             top,      logprobs,   entropy, lse,  top_ids,      top_logprobs, di.status, 0};
    auto st = static_cast<cudaStream_t>(stream);
    if (type == LAYA_TYPE_F32) return logprobs_go<float>(p, di.sms, st);
    if (type == LAYA_TYPE_F16) return logprobs_go<half>(p, di.sms, st);
    return logprobs_go<__nv_bfloat16>(p, di.sms, st);
  });
}
