// Attention of a batch whose sequences share a prefix.
//
// A query row's keys are the prefix's and its own sequence's:
//   o = sum_k e^(s_k) v_k / sum_k e^(s_k),   s = scale q.k.
// The softmax over a union of key sets joins from each set's normalised
// output o_s and l_s = log2 sum 2^(s_k log2 e):
//   l = log2 sum_s 2^(l_s),   o = sum_s 2^(l_s - l) o_s,
// so the prefix is one attention of all rows of the batch against one key
// list (read once, not once per sequence), each sequence's own keys another,
// and the partial results (F32) are joined.
//
// Launches: the prefix kernel and the own-keys kernel write partials (the
// second starts as the first's CTAs leave their SMs, programmatic dependent
// launch), and a third joins them; without a prefix, and with own keys that
// are not split, the own-keys kernel writes the output itself.  (Joining in
// the own-keys kernel, behind its pages, was slower: its few rows per CTA
// expose the latency of every plane's load.  512 rows x 16384 keys x 32 heads
// of 128, with an earlier prefix kernel: 280 us against 230.)
//
// Figures in this file are GPU time per call, replayed from a CUDA graph in
// runs of a few ms at 1965 MHz; those in pairs compare builds that differ in
// what is described alone.  The present code: 512 rows x 16384 keys x 32/8
// heads of 128 in BF16 176 us (202 in long runs, which the power limit holds
// near 1640 MHz), 64 x 4001 x 28/4 of 128 22.5, 33 x 6000 x 8/2 of 256 27.1.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "device_ops.h"
#include "gemm.h"
#include "launch.h"
#include "mma.cuh"
#include "ptx.cuh"

namespace laya {

namespace {

constexpr long long kBudget = 400000000ll;  // SM cycles per bounded wait (~0.2 s)
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxKeys = 0x7fffffff - 63;

struct PfxParams {
  const void* q;
  long long q_stride;
  int rows, H, KV, G;
  const int* offsets;
  int n_seqs, max_q;
  const int* prefix_pages;
  int prefix_len;
  const int* tables;
  long long tstride;
  int width;
  const int* lens;
  float scale_log2;
  void* out;
  long long out_stride;
  float* lse;
  float* part_o;  // [splits][rows][H][HD]: prefix splits, then own-key splits
  float* part_l;  // [splits][rows][H], log2 units
  int sp, ss;     // most prefix splits of a row (0: no prefix), own-key splits
  int q_tiles;    // row tiles per sequence (own keys) or over all rows (prefix)
  // tensor-core prefix kernel (chunk > 0): its units (kv head, unit_tok tokens)
  // are `steps` pages each, cut into runs of `chunk` pages over all units
  int chunk, steps, unit_tok, n_units;
  int pages;      // pages of the cache
  unsigned* status;
};

template <typename E>
struct Mma;
template <>
struct Mma<half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma16816(d, a, b0, b1);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_h2(a, b); }
  static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<half2*>(&x)); }
};
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2 of a sum l of 2^(x - m2); -inf of an empty one, a NaN stays.
__device__ __forceinline__ float log2_sum(float m2, float l) { return l == 0.f ? -INFINITY : m2 + log2f(l); }

// Bits 15 and 31: the halves of two packed 16-bit values that are infinite or NaN.
template <typename E>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  return ((x & 0x7fff7fffu) + (__is_same(E, half) ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

__device__ __forceinline__ void st_global_8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
               "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// Byte offset of 16-byte piece c of row r in a [HD / 64 blocks][R rows][128 B]
// tile with 128-byte swizzle.
template <int R>
__device__ __forceinline__ int tile_off(int r, int c) {
  return (c >> 3) * (R * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// A sequence's rows and keys, its device-side sizes checked.
struct Seq {
  int q0, nq, len, keys;  // first row, rows (at most max_q), own tokens, own keys that its table holds
};
__device__ __forceinline__ Seq seq_of(const PfxParams& p, int b) {
  const int a = p.offsets[b], e = p.offsets[b + 1], l = p.lens[b];
  Seq s;
  s.q0 = min(max(a, 0), p.rows);
  const int n = min(max(e, s.q0), p.rows) - s.q0;
  s.nq = min(n, p.max_q);
  s.len = max(l, 0) - (n - s.nq);  // so that row j sees keys 0 .. len - nq + j whether or not rows were cut
  s.keys = (int)min((long long)max(l, 0), (long long)p.width * 64);
  return s;
}
__device__ __forceinline__ void check_seq(const PfxParams& p, int b) {
  const int a = p.offsets[b], e = p.offsets[b + 1], l = p.lens[b];
  unsigned bad = 0;
  if (a < 0 || e < a || e > p.rows || e - a > p.max_q) bad |= LAYA_STATUS_ROWS;
  if (l < 0 || (long long)l > (long long)p.width * 64) bad |= LAYA_STATUS_PAGE;
  if (bad) atomicOr(p.status, bad);
}

// Prefix splits of a row of token tok, kv head kvh.
__device__ __forceinline__ int prefix_splits(const PfxParams& p, int tok, int kvh) {
  if (!p.chunk || !p.sp) return p.sp;
  const int n_tp = p.n_units / p.KV;
  const long long u = kvh * n_tp + tok / p.unit_tok;
  return (int)(((u + 1) * p.steps - 1) / p.chunk - u * p.steps / p.chunk) + 1;
}

constexpr int kOwnRegs = 144;  // of the unit kernel, head_dim 64 and 128

template <int HD, bool SPLITK>
struct Unit {
  static constexpr int ROWS = SPLITK ? 16 : 64;
  static constexpr int PAGE = 64 * HD * 2;  // K or V of one page
  static constexpr int STAGE = 2 * PAGE;
  static constexpr int S = HD == 64 ? 4 : HD == 128 ? 2 : 3;
  // SPLITK: two warps share a page (32 keys each), PW pages are in work at a
  // time.  S is a multiple of PW, so a stage is always the same warps': a warp
  // that waited for another's stage could meet its barrier a phase early and
  // take the old phase for the new.
  static constexpr int PW = HD == 256 ? 3 : 2;
  static constexpr int NW = SPLITK ? 2 * PW : 4;
  static constexpr int KEYS = SPLITK ? 32 : 64;  // of a page per warp
  static constexpr int THREADS = 32 * NW;
  static constexpr int CTAS = HD == 256 ? 1 : HD == 128 && !SPLITK ? 2 : 3;  // per SM
  static constexpr int OFF_Q = S * STAGE;  // [HD / 64][ROWS][128 B]
  static constexpr int OFF_BAR = OFF_Q + ROWS * HD * 2;
  static constexpr int SMEM = OFF_BAR + 2 * S * 8 + S * 4 + 1024;
  static_assert(!SPLITK || S % PW == 0, "a stage belongs to the same warps");
  static_assert(CTAS * (SMEM + 1024) <= 233472, "shared memory per SM");
  static_assert(NW * 16 * (HD + 2) * 4 <= S * STAGE, "the states' merge fits the ring");
};

// Attention of a tile of query rows over a list of whole 64-token pages with
// mma.sync m16n8k16, for few rows per key list, where the K/V bytes bound it.
// Each page's K and V come by TMA (128-byte swizzled boxes) into a ring; the
// first warp of those that share a stage fills it again when they are done.
//   SPLITK: 16 rows; warps 2 w and 2 w + 1 take halves of pages w, w + PW, ...
//           with online softmaxes of their own, and the warps' states are joined
//           in shared memory.
//   else  : 64 rows; warp w has rows 16 w .. 16 w + 15 and sees every page.
// OWN: unit = (sequence, kv head, row tile, own-key split), rows flattened as
// token * G + head of the group; otherwise (kv head, row tile, prefix split)
// over all rows of the batch.
// A unit is short (a few pages), so its chain of latencies (sizes, page
// numbers, pages, partials, output) is hidden by other units: small rings,
// two or three CTAs per SM (us, against rings that fill an SM's shared memory
// and one CTA: 64 sequences of one row 25 / 31, 33 to 96 rows each 26 / 33, 512
// rows behind 16384 shared keys 180 / 243, where they also find room
// beside the prefix kernel).
template <typename E, int HD, bool SPLITK, bool OWN>
__global__ void __maxnreg__((HD == 256 ? 255 : kOwnRegs))
    prefix_unit_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const PfxParams p) {
  using C = Unit<HD, SPLITK>;
  constexpr int ROWS = C::ROWS;
  extern __shared__ uint8_t pu_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pu_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = sm + C::OFF_Q;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
  uint64_t* empty = full + C::S;
  int* page_ok = reinterpret_cast<int*>(empty + C::S);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  int u = blockIdx.x;
  const int splits = OWN ? p.ss : p.sp;
  const int split = u % splits;
  u /= splits;
  const int kvh = u % p.KV;
  u /= p.KV;
  const int tile = u % p.q_tiles, b = u / p.q_tiles;
  const int* list = OWN ? p.tables + (long long)b * p.tstride : p.prefix_pages;
  // The warps that share pages: SPLITK pairs (pages w, w + PW, ...), else all.
  constexpr int STEP = SPLITK ? C::PW : 1;
  const int first = SPLITK ? warp >> 1 : 0;
  const bool leads = (SPLITK ? (warp & 1) == 0 : warp == 0);
  // the first page numbers, before the sizes that say how many count
  const int list_len = OWN ? p.width : (p.prefix_len + 63) / 64;
  int ids = splits == 1 && lane < list_len ? list[lane] : 0;

  Seq sq;
  if (OWN) {
    sq = seq_of(p, b);
    if (tid == 0 && kvh == 0 && tile == 0 && split == 0) check_seq(p, b);
  } else {
    sq = {0, p.rows, p.prefix_len, p.prefix_len};
  }
  const int f0 = tile * ROWS, n_flat = sq.nq * p.G;
  const int nr = min(ROWS, n_flat - f0);  // rows of this tile
  if (nr <= 0) {
    if (OWN && blockIdx.x == 0) pdl_wait();  // as at the end
    return;
  }
  // keys that row f sees: OWN len - nq + token + 1 (may be < 1), else all
  const int first_vis = OWN ? sq.len - sq.nq + f0 / p.G + 1 : p.prefix_len;
  const int last_vis = min(sq.keys, OWN ? sq.len - sq.nq + (f0 + nr - 1) / p.G + 1 : p.prefix_len);
  const int n_pages = max(0, (last_vis + 63) / 64);
  const int per = (n_pages + splits - 1) / splits;
  const int p0 = min(n_pages, split * per), np = min(n_pages, p0 + per) - p0;

  if (tid == 0) {
    for (int i = 0; i < C::S; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], SPLITK ? 2 : 4);
    }
    mbar_fence_init();
  }
  // Q rows as [HD / 64][ROWS][128 B], swizzled; rows past the tile are zero
  for (int i = tid; i < ROWS * (HD / 8); i += C::THREADS) {
    const int r = i / (HD / 8), c = i % (HD / 8);
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < nr) {
      const int f = f0 + r;
      x = *reinterpret_cast<const uint4*>(static_cast<const E*>(p.q) + (long long)(sq.q0 + f / p.G) * p.q_stride +
                                          (kvh * p.G + f % p.G) * HD + c * 8);
    }
    *reinterpret_cast<uint4*>(sQ + tile_off<ROWS>(r, c)) = x;
  }
  __syncthreads();
  if (!OWN) pdl_trigger();

  const bool partial = !OWN || p.ss > 1 || p.sp > 0;
  const int plane = OWN ? p.sp + split : split;
  const size_t rowsH = (size_t)p.rows * p.H;
  const int g = lane >> 2, t = lane & 3;
  const int wr = SPLITK ? 0 : warp * 16;  // this warp's first row
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float acc[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;

  if (splits > 1) ids = p0 + lane < n_pages ? list[p0 + lane] : 0;
  // Page i of this CTA's into stage i % S: lane 0 of a leading warp, which its
  // stage's warps have left (or that holds nothing yet).
  auto fill = [&](int i) {
    const int page = i < 32 ? __shfl_sync(0xffffffffu, ids, i) : list[p0 + i];
    if (lane == 0) {
      const int st = i % C::S;
      const bool in = page >= 0 && page < p.pages;
      page_ok[st] = in;
      if (in) {
        uint8_t* dst = sm + st * C::STAGE;
        mbar_expect_tx(&full[st], C::STAGE);
#pragma unroll
        for (int hb = 0; hb < HD / 64; hb++) {
          tma_load_4d(dst + hb * 8192, &tk, &full[st], hb * 64, 0, kvh, page);
          tma_load_4d(dst + C::PAGE + hb * 8192, &tv, &full[st], hb * 64, 0, kvh, page);
        }
      } else {
        atomicOr(p.status, LAYA_STATUS_PAGE);
        mbar_arrive(&full[st]);
      }
    }
  };
  int filled = -1;  // the last page that this (leading) warp asked for
  if (leads)
    for (int i = first; i < min(np, C::S); i += STEP) fill(filled = i);
  bool live = true;  // false once a wait ran out; the warps keep to the same barriers
  // visible keys of this thread's two rows
  int vis[2];
#pragma unroll
  for (int h = 0; h < 2; h++)
    vis[h] = OWN ? min(sq.keys, sq.len - sq.nq + (f0 + wr + g + 8 * h) / p.G + 1) : p.prefix_len;
  constexpr int KEYS = C::KEYS;
  const int koff = SPLITK ? (warp & 1) * 32 : 0;  // this warp's first key of a page
  const int me = SPLITK ? lane : tid, sharers = SPLITK ? 32 : 128;  // threads that share those keys
  auto sync = [&] {
    if (SPLITK)
      __syncwarp();
    else
      __syncthreads();
  };
  for (int i = first; i < np; i += STEP) {
    const int st = i % C::S;
    if (live && !__all_sync(0xffffffffu, mbar_wait(&full[st], (i / C::S) & 1, kBudget))) {
      live = false;
      if (lane == 0) atomicOr(p.status, LAYA_STATUS_TIMEOUT);
    }
    const uint8_t* sK = sm + st * C::STAGE;
    uint8_t* sV = sm + st * C::STAGE + C::PAGE;
    const int key0 = (p0 + i) * 64;
    const bool ok = live && page_ok[st];
    float sc[KEYS / 8][4];
    if (ok) {
#pragma unroll
      for (int j = 0; j < KEYS / 8; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      const int mat = lane / 8;
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk++) {
        uint32_t qa[4];
        ldsm_x4(qa, sQ + tile_off<ROWS>(wr + (lane % 8) + (mat % 2) * 8, kk * 2 + mat / 2));
#pragma unroll
        for (int nj = 0; nj < KEYS / 8; nj += 2) {
          uint32_t bf[4];
          ldsm_x4(bf, sK + tile_off<64>(koff + nj * 8 + (lane % 8) + (mat / 2) * 8, kk * 2 + (mat % 2)));
          Mma<E>::run(sc[nj], qa, bf[0], bf[1]);
          Mma<E>::run(sc[nj + 1], qa, bf[2], bf[3]);
        }
      }
      if (key0 + 64 > min(first_vis, sq.keys)) {
#pragma unroll
        for (int j = 0; j < KEYS / 8; j++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (key0 + koff + j * 8 + 2 * t + (e & 1) >= vis[e >> 1]) sc[j][e] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < KEYS / 8; j++) mx = fmaxf(mx, fmaxf(sc[j][2 * h], sc[j][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[h], mx);
        // a row that has seen no key yet keeps reference 0: its terms are 2^-inf = 0
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2((m[h] - ref) * p.scale_log2), off = -ref * p.scale_log2;
        m[h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < KEYS / 8; j++) {
          sc[j][2 * h] = ex2(fmaf(sc[j][2 * h], p.scale_log2, off));
          sc[j][2 * h + 1] = ex2(fmaf(sc[j][2 * h + 1], p.scale_log2, off));
          sum += sc[j][2 * h] + sc[j][2 * h + 1];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        l[h] = l[h] * corr + sum;
#pragma unroll
        for (int d = 0; d < HD / 8; d++) {
          acc[d][2 * h] *= corr;
          acc[d][2 * h + 1] *= corr;
        }
      }
    }
    // A probability of 0 times NaN or infinity is NaN.  Keys that no row of the
    // tile sees may hold anything: their values become 0.
    const bool tail = key0 + 64 > last_vis;
    if (tail && ok) {
      const int from = max(last_vis - key0, koff);
      for (int x = me; x < (koff + KEYS - from) * (HD / 8); x += sharers)
        *reinterpret_cast<uint4*>(sV + tile_off<64>(from + x / (HD / 8), x % (HD / 8))) = make_uint4(0u, 0u, 0u, 0u);
    }
    // Keys that some of its rows see and some do not (later tokens of the
    // sequence): what is not finite is added to the rows that see it by hand
    // (any probability times it is itself) and leaves the page.
    const int lo = max(first_vis - key0, koff), hi = min(last_vis - key0, koff + KEYS);
    if (OWN && lo < hi) {
      bool odd = false;
      if (ok)
        for (int x = me; x < (hi - lo) * (HD / 8); x += sharers) {
          const uint4 w = *reinterpret_cast<const uint4*>(sV + tile_off<64>(lo + x / (HD / 8), x % (HD / 8)));
          odd |= (not_finite<E>(w.x) | not_finite<E>(w.y) | not_finite<E>(w.z) | not_finite<E>(w.w)) != 0;
        }
      if (SPLITK ? __any_sync(0xffffffffu, odd) : __syncthreads_or(odd)) {
        if (ok)
#pragma unroll 1
          for (int key = lo; key < hi; key++)
#pragma unroll
            for (int d = 0; d < HD / 8; d++) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(sV + tile_off<64>(key, d) + 4 * t);
              const uint32_t bad = not_finite<E>(w);
              const float2 v = Mma<E>::unpack(w);
#pragma unroll
              for (int h = 0; h < 2; h++)
                if (key0 + key < vis[h]) {
                  if (bad & 0x8000u) acc[d][2 * h] += v.x;
                  if (bad & 0x80000000u) acc[d][2 * h + 1] += v.y;
                }
            }
        sync();
        if (ok)
#pragma unroll 1
          for (int x = me; x < (hi - lo) * (HD / 2); x += sharers) {
            uint32_t* w = reinterpret_cast<uint32_t*>(sV + tile_off<64>(lo + x / (HD / 2), x % (HD / 2) / 4) + x % 4 * 4);
            const uint32_t bad = not_finite<E>(*w);
            *w &= ~((bad & 0x8000u ? 0xffffu : 0u) | (bad & 0x80000000u ? 0xffff0000u : 0u));
          }
        sync();
      } else if (SPLITK) {
        __syncwarp();
      }
    } else if (tail) {
      sync();
    }
    if (ok) {
      const int mat = lane / 8;
#pragma unroll
      for (int kk = 0; kk < KEYS / 16; kk++) {
        // probabilities rounded to the cache's type: the second product's operand
        const uint32_t pa[4] = {Mma<E>::pack(sc[2 * kk][0], sc[2 * kk][1]), Mma<E>::pack(sc[2 * kk][2], sc[2 * kk][3]),
                                Mma<E>::pack(sc[2 * kk + 1][0], sc[2 * kk + 1][1]),
                                Mma<E>::pack(sc[2 * kk + 1][2], sc[2 * kk + 1][3])};
#pragma unroll
        for (int nd = 0; nd < HD / 8; nd += 2) {
          uint32_t bf[4];
          ldsm_x4_t(bf, sV + tile_off<64>(koff + kk * 16 + (lane % 8) + (mat % 2) * 8, nd + mat / 2));
          Mma<E>::run(acc[nd], pa, bf[0], bf[1]);
          Mma<E>::run(acc[nd + 1], pa, bf[2], bf[3]);
        }
      }
    }
    __syncwarp();
    if (live && i + C::S < np) {  // the stage's next page, once its warps have left it
      if (lane == 0) mbar_arrive(&empty[st]);
      if (leads) {
        if (__all_sync(0xffffffffu, mbar_wait(&empty[st], (i / C::S) & 1, kBudget))) {
          fill(filled = i + C::S);
        } else {
          live = false;
          if (lane == 0) atomicOr(p.status, LAYA_STATUS_TIMEOUT);
        }
      }
    }
  }
  // after a timeout: the copies that are still on their way land before the ring is used again
  if (!live && leads)
    for (int x = filled; x >= 0 && x > filled - C::S; x -= STEP) mbar_wait(&full[x % C::S], (x / C::S) & 1, kBudget);
  // ---- the tile's results
  if constexpr (SPLITK) {
    // join the warps' states through the (drained) ring: [NW][16][HD + 2]
    __syncthreads();
    float* comb = reinterpret_cast<float*>(sm);
    {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float* cw = comb + (warp * 16 + g + 8 * h) * (HD + 2);
        if (t == 0) {
          cw[0] = m[h] * p.scale_log2;
          cw[1] = l[h];
        }
#pragma unroll
        for (int d = 0; d < HD / 8; d++)
          *reinterpret_cast<float2*>(cw + 2 + d * 8 + 2 * t) = make_float2(acc[d][2 * h], acc[d][2 * h + 1]);
      }
    }
    __syncthreads();
    for (int i = tid; i < nr * (HD / 2); i += C::THREADS) {
      const int r = i / (HD / 2), d = (i % (HD / 2)) * 2;
      const int f = f0 + r, tok = sq.q0 + f / p.G, h = kvh * p.G + f % p.G;
      const size_t th = (size_t)tok * p.H + h;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < C::NW; w++) M = fmaxf(M, comb[(w * 16 + r) * (HD + 2)]);
      const float ref = M == -INFINITY ? 0.f : M;
      float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int w = 0; w < C::NW; w++) {
        const float* cw = comb + (w * 16 + r) * (HD + 2);
        const float wt = ex2(cw[0] - ref);
        const float2 x = *reinterpret_cast<const float2*>(cw + 2 + d);
        sum = fmaf(wt, cw[1], sum);
        v0 = fmaf(wt, x.x, v0);
        v1 = fmaf(wt, x.y, v1);
      }
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
      const float l2 = log2_sum(M, sum);
      if (partial) {
        if (d == 0) p.part_l[plane * rowsH + th] = l2;
        *reinterpret_cast<float2*>(p.part_o + (plane * rowsH + th) * HD + d) = make_float2(v0 * inv, v1 * inv);
      } else {
        if (d == 0 && p.lse) p.lse[th] = l2 * kLn2;
        *reinterpret_cast<uint32_t*>(static_cast<E*>(p.out) + (long long)tok * p.out_stride + h * HD + d) =
            Mma<E>::pack(v0 * inv, v1 * inv);
      }
    }
  } else {
    {
#pragma unroll
      for (int hh = 0; hh < 2; hh++) {
        const int r = wr + g + 8 * hh;
        if (r >= nr) continue;
        const int f = f0 + r, tok = sq.q0 + f / p.G, h = kvh * p.G + f % p.G;
        const size_t th = (size_t)tok * p.H + h;
        const float inv = l[hh] > 0.f || l[hh] != l[hh] ? 1.f / l[hh] : 0.f;
        const float l2 = log2_sum(m[hh] * p.scale_log2, l[hh]);
        if (partial) {
          if (t == 0) p.part_l[plane * rowsH + th] = l2;
#pragma unroll
          for (int d = 0; d < HD / 8; d++)
            *reinterpret_cast<float2*>(p.part_o + (plane * rowsH + th) * HD + d * 8 + 2 * t) =
                make_float2(acc[d][2 * hh] * inv, acc[d][2 * hh + 1] * inv);
        } else {
          if (t == 0 && p.lse) p.lse[th] = l2 * kLn2;
          E* dst = static_cast<E*>(p.out) + (long long)tok * p.out_stride + h * HD + 2 * t;
#pragma unroll
          for (int d = 0; d < HD / 8; d++)
            *reinterpret_cast<uint32_t*>(dst + d * 8) = Mma<E>::pack(acc[d][2 * hh] * inv, acc[d][2 * hh + 1] * inv);
        }
      }
    }
  }
  // The join kernel's griddepcontrol.wait has to cover the prefix kernel, too:
  // one CTA ends after it, and with that this kernel does (all of them would
  // keep their places on the SMs).
  if (OWN && blockIdx.x == 0) pdl_wait();
}

// ------------------------------------------------------------ prefix, many rows
//
// For more than 16 rows per kv head the prefix is a product of matrices and
// runs on the tcgen05 tensor cores.  A unit is one kv head and NT tiles of
// 128 query rows (a tile: TT = 128 / G tokens, row = token * G + head of the
// group); its keys go by a page (64) at a time:
//   S = Q K^T   (M 128, N 64, into one of the tile's two score buffers in TMEM),
//   P = 2^(S - ref),  O += P V
// with P written back over S in TMEM as the next product's A operand.
//   warp 0        TMA: Q, then K and V of each page into one ring of stages, in
//                 the order of the products
//   warp 1        one thread issues the products, the scores two pages ahead:
//                 the softmax of a page does not wait for its scores
//   warps 4 ..    softmax, four warps per tile, thread = row = TMEM lane.  O is
//                 rescaled in TMEM only when a row's maximum passes its
//                 reference by 2^15 (P stays below 2^15; ref = max - 7 keeps
//                 small probabilities out of F16's subnormals).
// Per page and two tiles at head_dim 128 the tensor cores need 1024 cycles (the
// scores' N = 64 makes shared memory their limit: 1280) and the exponentials
// (16384 at 16 per cycle) 1024, so both have to run at once.  With one score
// buffer of 128 keys per tile, scores issued behind the page's P V, they took
// turns (51% and 52% busy; eight softmax warps per tile changed nothing).
// Two tiles per unit halve the K/V bytes from L2 per row; head_dim 256 has room
// for one tile in TMEM.
// The pages of all units, one unit after the other, are cut into equal runs,
// one per CTA, so the GPU is evenly loaded whatever the sizes; a unit cut by a
// run's end leaves one partial result per run (prefix_splits).
// The last page's rows past the prefix come as zeros from a tensor map that
// ends there, so nothing stale meets a probability of 0; pages outside the
// cache are loaded out of bounds (zeros) and masked.
template <int HD, int NT_>
struct Ptc {
  static constexpr int NT = NT_;
  static constexpr int Q_TILE = 128 * HD * 2;  // [HD / 64][128 rows][128 B]
  static constexpr int STAGE = 64 * HD * 2;    // K or V of a page: [HD / 64][64 rows][128 B]
  static constexpr int NS = HD == 256 ? 4 : HD == 64 ? (NT == 1 ? 9 : 10) : NT == 1 ? 3 : 5;
  static constexpr int OFF_RING = NT * Q_TILE;
  static constexpr int OFF_BAR = OFF_RING + NS * STAGE;
  static constexpr int SMEM = OFF_BAR + (2 * NS + 3 + 7 * NT) * 8 + 16 + 1024;
  static constexpr int THREADS = 128 + NT * 128;
  static constexpr int COLS = NT * (128 + HD) <= 256 ? 256 : 512;
  static constexpr int S_COL = 0, O_COL = NT * 128;  // tile t: S at 128 t and 128 t + 64, O at O_COL + HD t
  // Registers per thread and the ring's depth leave the own-keys kernel's CTAs
  // (a warp per SM quarter, kOwnRegs) room on the SM: one beside two tiles, two
  // beside one tile (64 rows, 4001 shared keys x 28/4 heads of 128: 21.4 us,
  // against 25 with six stages and one).  head_dim 256 has none anyway.
  static constexpr int REGS = 112;
  static constexpr int BESIDE = HD == 256 ? 0 : NT == 2 ? 1 : 2;
  static_assert(O_COL + NT * HD <= COLS, "TMEM columns");
  static_assert(SMEM <= 232448, "shared memory per CTA");
  static_assert(SMEM + 1024 + BESIDE * (Unit<HD, true>::SMEM + 1024) <= 233472, "shared memory per SM");
  static_assert((THREADS / 128 * REGS + BESIDE * kOwnRegs) * 32 <= 16384, "registers per SM quarter");
};


struct Run {  // a CTA's part of a unit: pages s0 .. s1 - 1
  int kvh, tok0, s0, s1, plane, tiles;
};

// The next part of a CTA's run [c * chunk, (c + 1) * chunk) of pages.
__device__ __forceinline__ bool run_part(const PfxParams& p, long long& at, long long end, int nt, int tt, Run& r) {
  if (at >= end) return false;
  const long long u = at / p.steps;
  const int n_tp = p.n_units / p.KV;
  r.kvh = (int)(u / n_tp);
  r.tok0 = (int)(u % n_tp) * p.unit_tok;
  r.s0 = (int)(at - u * p.steps);
  r.s1 = (int)min((long long)p.steps, r.s0 + (end - at));
  r.plane = (int)(at / p.chunk - u * p.steps / p.chunk);
  r.tiles = min(nt, (p.rows - r.tok0 + tt - 1) / tt);
  at += r.s1 - r.s0;
  return true;
}

template <typename E, int HD, int NT>
__global__ void __maxnreg__((Ptc<HD, NT>::REGS))
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tv_last,
                     const PfxParams p) {
  using C = Ptc<HD, NT>;
  extern __shared__ uint8_t pt_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sm + C::OFF_RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);  // [NS]
  uint64_t* empty = full + C::NS;                                 // [NS]
  uint64_t* q_full = empty + C::NS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;      // [NT][2] scores of a page
  uint64_t* p_full = s_full + 2 * NT;  // [NT][2] probabilities of a page (4 warps)
  uint64_t* o_done = p_full + 2 * NT;  // [NT] one phase per page's P V
  uint64_t* o_full = o_done + NT;      // [NT] O of a part complete
  uint64_t* o_empty = o_full + NT;     // [NT] O read (4 warps)
  uint64_t* fin = o_empty + NT;        // all products of the CTA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = p.G, TT = 128 / G;
  // tile rows that no token has (G not a divisor of 128) are zero: finite scores, never written out
  for (int i = threadIdx.x; i < NT * (HD / 64) * (128 - TT * G) * 8; i += C::THREADS) {
    const int per = (128 - TT * G) * 8, blk = i / per, e = i % per;
    reinterpret_cast<uint4*>(sm + blk * 16384 + TT * G * 128)[e] = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_async_smem();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NS; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(fin, 1);
    for (int t = 0; t < NT; t++) {
      for (int i = 0; i < 2; i++) {
        mbar_init(&s_full[2 * t + i], 1);
        mbar_init(&p_full[2 * t + i], 4);
      }
      mbar_init(&o_done[t], 1);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 4);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tbase = *tmem_slot;
  long long at = (long long)blockIdx.x * p.chunk;
  const long long end = min(at + p.chunk, (long long)p.n_units * p.steps);
  unsigned bad = 0;
  bool live = true;  // false once a wait ran out: every role then leaves its loops
  auto wait = [&](uint64_t* b, uint32_t parity) {
    if (live && !mbar_wait(b, parity, kBudget)) live = false;
    return live;
  };
  Run r;

  if (warp < 4) {
    if (warp == 0) {
      if (lane == 0) {
        int g = 0, k = 0;  // stages, parts
        while (live && run_part(p, at, end, NT, TT, r)) {
          if (!wait(q_empty, (k & 1) ^ 1)) break;
          mbar_expect_tx(q_full, (uint32_t)(r.tiles * TT * G * 128 * (HD / 64)));
          for (int t = 0; t < r.tiles; t++)
#pragma unroll
            for (int hb = 0; hb < HD / 64; hb++)
              tma_load_3d(sm + t * C::Q_TILE + hb * 16384, &tq, q_full, hb * 64, r.kvh * G, r.tok0 + t * TT);
          k++;
          // in the order of use: K 0, K 1, V 0, K 2, V 1, ..., the last V
          const int ns = r.s1 - r.s0;
          int page_k = p.prefix_pages[r.s0], page_v[2] = {0, 0};  // of the next K, and of the V that are behind it
          for (int x = 0, jk = 0, jv = 0; x < 2 * ns && live; x++) {
            const bool is_k = jk < min(ns, jv + 2);
            int page;
            if (is_k) {
              page = page_k;
              if (++jk < ns) page_k = p.prefix_pages[r.s0 + jk];
              if (page < 0 || page >= p.pages) {
                bad |= LAYA_STATUS_PAGE;
                page = p.pages;  // out of bounds: zeros
              }
              page_v[0] = page_v[1];
              page_v[1] = page;
            } else {
              page = jk - jv == 2 ? page_v[0] : page_v[1];
              jv++;
            }
            const int st = g % C::NS;
            if (!wait(&empty[st], ((g / C::NS) & 1) ^ 1)) break;
            g++;
            mbar_expect_tx(&full[st], C::STAGE);
            const void* map = is_k ? &tk : r.s0 + jv == p.steps ? &tv_last : &tv;
#pragma unroll
            for (int hb = 0; hb < HD / 64; hb++)
              tma_load_4d(ring + st * C::STAGE + hb * 8192, map, &full[st], hb * 64, 0, r.kvh, page);
          }
        }
        // the last use of every stage is over, or after a timeout its copy has
        // landed, before the CTA may end
        for (int x = max(0, g - C::NS); x < g; x++)
          if (!wait(&empty[x % C::NS], (x / C::NS) & 1)) mbar_wait(&full[x % C::NS], (x / C::NS) & 1, kBudget);
        if (!live && k) mbar_wait(q_full, (k - 1) & 1, kBudget);
      }
    } else if (warp == 1) {
      if (elect_one()) {
        constexpr bool BF = !__is_same(E, half);
        const uint32_t id_s = BF ? idesc_bf16_f32(128, 64) : idesc_f16_f32(128, 64);
        const uint32_t id_o = (BF ? idesc_bf16_f32(128, HD) : idesc_f16_f32(128, HD)) | (1u << 16);  // V MN-major
        int g = 0, k = 0;
        int steps_t[NT] = {}, parts_t[NT] = {};  // pages with P V issued, parts, of each tile
        while (live && run_part(p, at, end, NT, TT, r)) {
          if (!wait(q_full, k & 1)) break;
          k++;
          const int ns = r.s1 - r.s0;
          // scores of the part's page j for tile t
          auto scores = [&](int j, int t) {
            const int x = g + j + max(0, j - 1), st = x % C::NS, buf = (steps_t[t] + (j > 1 ? 1 : j)) & 1;
            if (!wait(&full[st], (x / C::NS) & 1)) return;
            tc_fence_after();
            // descriptors of the later k-steps: the start address field plus a constant
            const uint64_t qd = sw128_desc(smem_u32(sm + t * C::Q_TILE));
            const uint64_t kd = sw128_desc(smem_u32(ring + st * C::STAGE));
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++)
              umma_f16(tbase + C::S_COL + t * 128 + buf * 64, qd + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                       kd + (((kk >> 2) * 8192 + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[2 * t + buf]);
            if (t == r.tiles - 1) {
              umma_commit(&empty[st]);
              if (j == ns - 1) umma_commit(q_empty);
            }
          };
          for (int j = 0; j < 2 && j < ns; j++)
            for (int t = 0; t < r.tiles; t++) scores(j, t);
          for (int j = 0; j < ns && live; j++) {
            const int x = g + j + min(ns, j + 2), st = x % C::NS;
            for (int t = 0; t < r.tiles; t++) {
              const int buf = steps_t[t] & 1;
              if (j == 0) wait(&o_empty[t], (parts_t[t] & 1) ^ 1);
              wait(&full[st], (x / C::NS) & 1);
              if (!wait(&p_full[2 * t + buf], (steps_t[t] >> 1) & 1)) break;
              steps_t[t]++;
              tc_fence_after();
              const uint64_t vd = sw128_mn_desc(smem_u32(ring + st * C::STAGE), 8192, 1024);
#pragma unroll
              for (int kk = 0; kk < 4; kk++)
                umma_f16_ta(tbase + C::O_COL + t * HD, tbase + C::S_COL + t * 128 + buf * 64 + kk * 8,
                            vd + kk * (2048 >> 4), id_o, (j > 0 || kk > 0) ? 1u : 0u);
              umma_commit(&o_done[t]);
              if (t == r.tiles - 1) umma_commit(&empty[st]);
              if (j == ns - 1) {
                umma_commit(&o_full[t]);
                parts_t[t]++;
              }
              // over the P just used: products run in the order of issue
              if (j + 2 < ns) scores(j + 2, t);
            }
          }
          g += 2 * ns;
        }
        // every product is over before TMEM is freed
        umma_commit(fin);
        mbar_wait(fin, 0, kBudget);
      }
    }  // warps 2 and 3: nothing (a softmax warp's lanes go by warp % 4)
  } else {
    const int t = (warp - 4) / 4, quarter = warp % 4, row = quarter * 32 + lane;
    const uint32_t tl = tbase + ((uint32_t)(quarter * 32) << 16);
    const uint32_t tS = tl + C::S_COL + t * 128, tO = tl + C::O_COL + t * HD;
    int step = 0, part = 0;  // of this tile
    while (live && run_part(p, at, end, NT, TT, r)) {
      if (t >= r.tiles) continue;
      const int tok = r.tok0 + t * TT + row / G, h = r.kvh * G + row % G;
      const bool valid = row < TT * G && tok < p.rows;
      const bool busy = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps the barriers' count
      float mref = -INFINITY, l = 0.f;
      int next = __ldg(p.prefix_pages + r.s0);
      for (int s = r.s0; s < r.s1; s++, step++) {
        const int page = next, buf = step & 1;
        if (s + 1 < r.s1) next = __ldg(p.prefix_pages + s + 1);
        // keys of the page that are there
        const int seen = page >= 0 && page < p.pages ? min(64, p.prefix_len - s * 64) : 0;
        live = __all_sync(0xffffffffu, wait(&s_full[2 * t + buf], (step >> 1) & 1));
        if (!live) break;
        tc_fence_after();
        if (busy) {
          uint32_t v[64];
          __syncwarp();
          tmem_ld32(tS + buf * 64, *reinterpret_cast<uint32_t(*)[32]>(v));
          tmem_ld32(tS + buf * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
          tmem_ld_wait();
          if (seen < 64) {
#pragma unroll
            for (int c = 0; c < 64; c++)
              if (c >= seen) v[c] = 0xff800000u;
          }
          float m4[4];
#pragma unroll
          for (int c = 0; c < 4; c++) m4[c] = __uint_as_float(v[c]);
#pragma unroll
          for (int c = 4; c < 64; c++) m4[c & 3] = fmaxf(m4[c & 3], __uint_as_float(v[c]));
          // the scale is positive, so the maximum commutes with it
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
          const float nref = mx > mref + 15.f ? mx - 7.f : mref;
          if (s > r.s0 && __any_sync(0xffffffffu, nref != mref)) {
            // These scores were issued behind the P V before the last one, so
            // o_done is in the last one's phase or past it.
            live = __all_sync(0xffffffffu, wait(&o_done[t], (step - 1) & 1));
            if (!live) break;
            tc_fence_after();
            const float corr = nref != mref ? ex2(mref - nref) : 1.f;
#pragma unroll 1
            for (int c = 0; c < HD / 16; c++) {
              uint32_t o[16];
              __syncwarp();
              tmem_ld16(tO + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st16(tO + c * 16, o);
            }
            l *= corr;
          }
          mref = nref;
          unsigned long long sc2, nm2, acc2[2];
          const float off = mref == -INFINITY ? 0.f : -mref;  // nothing seen yet: every term is 2^-inf
          asm("mov.b64 %0, {%1, %1};" : "=l"(sc2) : "f"(p.scale_log2));
          asm("mov.b64 %0, {%1, %1};" : "=l"(nm2) : "f"(off));
          asm("mov.b64 %0, {%1, %1};" : "=l"(acc2[0]) : "f"(0.f));
          acc2[1] = acc2[0];
#pragma unroll
          for (int q = 0; q < 2; q++) {
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              unsigned long long x2, e2, p2;
              asm("mov.b64 %0, {%1, %2};" : "=l"(x2) : "r"(v[32 * q + c]), "r"(v[32 * q + c + 1]));
              asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e2) : "l"(x2), "l"(sc2), "l"(nm2));
              float e0, e1;
              asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(e2));
              e0 = ex2(e0);
              e1 = ex2(e1);
              asm("mov.b64 %0, {%1, %2};" : "=l"(p2) : "f"(e0), "f"(e1));
              asm("add.rn.f32x2 %0, %1, %2;" : "=l"(acc2[(c >> 1) & 1]) : "l"(acc2[(c >> 1) & 1]), "l"(p2));
              // rounded to the cache's type, the second product's operand
              w[c >> 1] = Mma<E>::pack(e0, e1);
            }
            __syncwarp();
            tmem_st16(tS + buf * 64 + q * 16, w);
          }
          float l4[4];
          asm("mov.b64 {%0, %1}, %2;" : "=f"(l4[0]), "=f"(l4[1]) : "l"(acc2[0]));
          asm("mov.b64 {%0, %1}, %2;" : "=f"(l4[2]), "=f"(l4[3]) : "l"(acc2[1]));
          l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + buf]);
      }
      if (!live) break;
      live = __all_sync(0xffffffffu, wait(&o_full[t], part & 1));
      if (!live) break;
      part++;
      tc_fence_after();
      if (busy) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const size_t th = (size_t)tok * p.H + h, rowsH = (size_t)p.rows * p.H;
        if (valid) p.part_l[r.plane * rowsH + th] = log2_sum(mref, l);
        // a lane holds a row: 32 bytes, a whole sector, per store
        float* dst = p.part_o + (r.plane * rowsH + th) * HD;
#pragma unroll 1
        for (int c = 0; c < HD / 32; c++) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait();
          if (valid) {
#pragma unroll
            for (int b = 0; b < 32; b += 8) {
              float x[8];
#pragma unroll
              for (int i = 0; i < 8; i++) x[i] = __uint_as_float(o[b + i]) * inv;
              st_global_8(dst + c * 32 + b, x);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[t]);
    }
  }
  if (!live) bad |= LAYA_STATUS_TIMEOUT;
  if (bad) atomicOr(p.status, bad);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, C::COLS);
  }
}

// Joins all partials of a row: prefix splits and own-key splits.  HD / 8
// lanes per row (token, head), eight values each, the loads of four planes in
// flight together; WAYS such groups share a row's planes where there are few
// rows, and meet in shared memory.  CTA = (sequence, 256 / (HD / 8) / WAYS of
// its rows).  Bound by latency (sizes, l_s, partials: dependent loads) and by
// the partials' bytes, which are in L2.
template <typename E, int HD, int WAYS>
__global__ void __launch_bounds__(256) prefix_join_kernel(const PfxParams p, int blocks_per_seq) {
  constexpr int L = HD / 8, R = 256 / L;  // lanes per group, groups per CTA
  const int b = blockIdx.x / blocks_per_seq, grp = threadIdx.x / L, way = grp % WAYS;
  const int i0 = (blockIdx.x % blocks_per_seq) * (R / WAYS) + grp / WAYS;
  const int sub = threadIdx.x % L;
  const Seq s = seq_of(p, b);
  pdl_wait();
  const bool in = i0 < s.nq * p.H;
  if (WAYS == 1 && !in) return;
  const int h = in ? i0 % p.H : 0, tok = in ? s.q0 + i0 / p.H : 0;
  const size_t rowsH = (size_t)p.rows * p.H, th = (size_t)tok * p.H + h;
  // planes 0 .. pre - 1 and sp .. sp + ss - 1
  const int pre = p.sp ? prefix_splits(p, tok, h / p.G) : 0, planes = in ? pre + p.ss : 0, gap = p.sp - pre;
  const float* pl = p.part_l + th;
  const float* po = p.part_o + th * HD + sub * 8;
  float M = -INFINITY, sum = 0.f, acc[8];
#pragma unroll
  for (int d = 0; d < 8; d++) acc[d] = 0.f;
  for (int j = way; j < planes; j += 4 * WAYS) {
    float li[4], x[4][8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = min(j + e * WAYS, planes - 1);
      const size_t plane = (i < pre ? i : i + gap) * rowsH;
      li[e] = j + e * WAYS < planes ? pl[plane] : -INFINITY;
      const float4 y = *reinterpret_cast<const float4*>(po + plane * HD);
      const float4 z = *reinterpret_cast<const float4*>(po + plane * HD + 4);
      x[e][0] = y.x, x[e][1] = y.y, x[e][2] = y.z, x[e][3] = y.w;
      x[e][4] = z.x, x[e][5] = z.y, x[e][6] = z.z, x[e][7] = z.w;
    }
    const float mn = fmaxf(M, fmaxf(fmaxf(li[0], li[1]), fmaxf(li[2], li[3])));
    const float ref = mn == -INFINITY ? 0.f : mn, corr = ex2(M - ref);
    M = mn;
    sum *= corr;
#pragma unroll
    for (int d = 0; d < 8; d++) acc[d] *= corr;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float wt = ex2(li[e] - ref);
      sum += wt;
#pragma unroll
      for (int d = 0; d < 8; d++) acc[d] = fmaf(wt, x[e][d], acc[d]);
    }
  }
  if constexpr (WAYS > 1) {
    __shared__ float meet[10][256];
    if (way) {
      meet[0][threadIdx.x] = M;
      meet[1][threadIdx.x] = sum;
#pragma unroll
      for (int d = 0; d < 8; d++) meet[2 + d][threadIdx.x] = acc[d];
    }
    __syncthreads();
    if (way) return;
#pragma unroll 1
    for (int w = 1; w < WAYS; w++) {
      const int at = threadIdx.x + w * L;
      const float mw = meet[0][at], mn = fmaxf(M, mw);
      const float ref = mn == -INFINITY ? 0.f : mn, c0 = ex2(M - ref), c1 = ex2(mw - ref);
      M = mn;
      sum = sum * c0 + meet[1][at] * c1;
#pragma unroll
      for (int d = 0; d < 8; d++) acc[d] = acc[d] * c0 + meet[2 + d][at] * c1;
    }
  }
  if (!in) return;
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (p.lse && sub == 0) p.lse[th] = log2_sum(M, sum) * kLn2;
  *reinterpret_cast<uint4*>(static_cast<E*>(p.out) + (long long)tok * p.out_stride + h * HD + sub * 8) =
      make_uint4(Mma<E>::pack(acc[0] * inv, acc[1] * inv), Mma<E>::pack(acc[2] * inv, acc[3] * inv),
                 Mma<E>::pack(acc[4] * inv, acc[5] * inv), Mma<E>::pack(acc[6] * inv, acc[7] * inv));
}

// ------------------------------------------------------------ host

// What a call's sizes decide: key splits and row tiles.
struct Shape {
  int sp, ss;      // most prefix splits of a row, own-key splits
  bool own_split;  // own keys: 16-row tiles with the pages shared by the warps
  int own_tiles, pre_tiles;
  bool tc;         // prefix on the tensor cores (else one 16-row tile per kv head)
  int nt;          // its tiles per CTA
  int chunk, steps, unit_tok, n_units, grid;
};

Shape shape_of(const laya_kv_pages& c, const laya_prefix_args& a, int sms) {
  Shape s{};
  const int G = a.heads / c.kv_heads;
  // no sequence has more rows than there are, however loose the caller's bound
  const long long flat = (long long)a.rows * G, own_flat = (long long)std::min(a.max_q, a.rows) * G;
  s.own_split = own_flat <= 16;
  s.own_tiles = (int)((own_flat + (s.own_split ? 16 : 64) - 1) / (s.own_split ? 16 : 64));
  const int pre_pages = (a.prefix_len + 63) / 64;
  s.pre_tiles = (int)((flat + 15) / 16);
  // 16-row tiles on mma.sync read the prefix once per tile, but start and end
  // sooner than the tensor-core kernel, which takes over at about ten tile-pages
  // of head_dim 64 per SM.  The square of head_dim counts: a tile's work per page
  // and how few CTAs an SM holds (us, mma.sync / tcgen05, tile-pages per
  // SM: 32 x 1000 keys x 32/8 heads of 64 11.1 / 12.2 at 7, 16 x 4000 14.7 / 13.7
  // at 14; 4 x 2000 x 28/4 of 128 10.6 / 11.1 at 1.7, 16 x 1000 12.8 / 11.1 at 3;
  // 16 x 1500 x 8/2 of 256 16.2 / 12.0 at 1.3).
  const long long wide = c.head_dim / 64;
  s.tc = flat > 16 && (long long)s.pre_tiles * c.kv_heads * pre_pages * wide * wide > 10ll * sms;
  if (pre_pages && !s.tc) {
    // Key splits until the CTAs fill the GPU once, at least two pages each.
    s.sp = (int)std::max(
        1ll, std::min<long long>(sms / std::max(1ll, (long long)c.kv_heads * s.pre_tiles), (pre_pages + 1) / 2));
  } else if (pre_pages) {
    s.steps = pre_pages;
    // Two tiles per CTA where a CTA has work for a while; one where it has
    // sixteen pages or fewer (us, one / two: 80 rows x 4000 keys x 28/4 heads of
    // 128 20.2 / 25.4, 160 rows 30.9 / 31.9, 640 rows x 1024 x 32/8 of 64 27.9 /
    // 25.5, 64 rows x 16000 42 / 36).
    const long long tiles = (a.rows + 128 / G - 1) / (128 / G);
    s.nt = c.head_dim == 256 || tiles * c.kv_heads * pre_pages <= 16ll * sms ? 1 : 2;
    s.unit_tok = s.nt * (128 / G);
    s.n_units = c.kv_heads * ((a.rows + s.unit_tok - 1) / s.unit_tok);
    const long long work = (long long)s.n_units * s.steps;
    s.chunk = (int)std::max(1ll, (work + sms - 1) / sms);
    s.grid = (int)((work + s.chunk - 1) / s.chunk);
    // a unit of `steps` touches at most this many runs of `chunk`
    s.sp = (s.steps - 2 + s.chunk) / s.chunk + 1;
  }
  const long long own_units = (long long)a.n_seqs * s.own_tiles * c.kv_heads;
  s.ss = (int)std::max(1ll, std::min<long long>(sms / std::max(1ll, own_units), (a.width + 7) / 8));
  return s;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

size_t workspace_of(const laya_kv_pages& c, const laya_prefix_args& a, const Shape& s) {
  const size_t planes = s.sp || s.ss > 1 ? s.sp + s.ss : 0, rowsH = (size_t)a.rows * a.heads;
  return align256(planes * rowsH * 4) + align256(planes * rowsH * c.head_dim * 4);
}

int check_sizes(const laya_kv_pages* c, const laya_prefix_args* a) {
  if (int rc = check_pages(c)) return rc;
  if (!a) return fail(LAYA_E_INVALID, "null argument");
  if (a->rows < 0 || a->n_seqs < 0 || a->max_q < 0 || a->prefix_len < 0 || a->width < 0)
    return fail(LAYA_E_INVALID, "negative size");
  if (a->heads < 1 || a->heads % c->kv_heads) return fail(LAYA_E_INVALID, "heads must be a multiple of kv_heads");
  if (a->heads / c->kv_heads > 128) return fail(LAYA_E_INVALID, "more than 128 query heads per kv head");
  if ((long long)a->rows * a->heads > 0x7fffffffll) return fail(LAYA_E_INVALID, "too many query rows");
  // positions up to the end of the last page are 32-bit
  if (a->prefix_len > kMaxKeys || a->width > kMaxKeys / 64)
    return fail(LAYA_E_INVALID, "prefix_len or width beyond 2^31 - 64 keys");
  return 0;
}

template <typename E, int HD, bool SPLITK, bool OWN>
int launch_unit(const CUtensorMap& tk, const CUtensorMap& tv, const PfxParams& p, long long grid, int dev, bool pdl,
                cudaStream_t st) {
  static std::atomic<bool> configured[64];
  if (!configured[dev & 63]) {
    LAYA_CK(cudaFuncSetAttribute(prefix_unit_kernel<E, HD, SPLITK, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 Unit<HD, SPLITK>::SMEM));
    LAYA_CK(cudaFuncSetAttribute(prefix_unit_kernel<E, HD, SPLITK, OWN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared));
    configured[dev & 63] = true;
  }
  if (grid > 0x7fffffffll) return fail(LAYA_E_INVALID, "too many attention units");
  LAYA_CK(launch_k(prefix_unit_kernel<E, HD, SPLITK, OWN>, dim3((unsigned)grid), dim3(Unit<HD, SPLITK>::THREADS), (size_t)Unit<HD, SPLITK>::SMEM, st,
                   pdl, tk, tv, p));
  return 0;
}

template <typename E, int HD, int NT>
int launch_tc(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tv_last,
              const PfxParams& p, int grid, int dev, cudaStream_t st) {
  using C = Ptc<HD, NT>;
  static std::atomic<bool> configured[64];
  if (!configured[dev & 63]) {
    LAYA_CK(cudaFuncSetAttribute(prefix_tc_kernel<E, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    LAYA_CK(cudaFuncSetAttribute(prefix_tc_kernel<E, HD, NT>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared));
    configured[dev & 63] = true;
  }
  LAYA_CK(launch_k(prefix_tc_kernel<E, HD, NT>, dim3(grid), dim3(C::THREADS), (size_t)C::SMEM, st, false, tq, tk, tv,
                   tv_last, p));
  return 0;
}

template <typename E, int HD>
int prefix_go(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tv_last, PfxParams p, const Shape& s, int dev, int sms,
              cudaStream_t st) {
  if (s.sp && !s.tc) {
    p.q_tiles = s.pre_tiles;
    if (int rc = launch_unit<E, HD, true, false>(tk, tv, p, (long long)p.KV * s.pre_tiles * s.sp, dev, false, st))
      return rc;
  } else if (s.sp) {
    int rc;
    if constexpr (HD == 256)
      rc = launch_tc<E, HD, 1>(tq, tk, tv, tv_last, p, s.grid, dev, st);
    else
      rc = s.nt == 1 ? launch_tc<E, HD, 1>(tq, tk, tv, tv_last, p, s.grid, dev, st)
                     : launch_tc<E, HD, 2>(tq, tk, tv, tv_last, p, s.grid, dev, st);
    if (rc) return rc;
  }
  p.q_tiles = s.own_tiles;
  const long long grid = (long long)p.n_seqs * s.own_tiles * p.KV * s.ss;
  if (int rc = s.own_split ? launch_unit<E, HD, true, true>(tk, tv, p, grid, dev, s.sp > 0, st)
                           : launch_unit<E, HD, false, true>(tk, tv, p, grid, dev, s.sp > 0, st))
    return rc;
  if (s.ss > 1 || s.sp) {
    // Eight groups per row where that saves a few rounds and the GPU holds the
    // CTAs (4 per SM) at once: 33 rows x 8 heads of 256, 34 planes 33.6 -> 29 us
    // a call; 64 x 28 of 128, 12 planes 26.2 -> 29.
    const int groups = 256 / (HD / 8), planes = s.sp + s.ss;
    const long long flat = (long long)std::min(p.max_q, p.rows) * p.H;
    const bool shared = planes > 16 && flat * p.n_seqs * 8 <= 4ll * sms * groups;
    const long long blocks = (flat * (shared ? 8 : 1) + groups - 1) / groups;
    if (blocks * p.n_seqs > 0x7fffffffll) return fail(LAYA_E_INVALID, "too many attention rows");
    LAYA_CK(launch_k(shared ? prefix_join_kernel<E, HD, 8> : prefix_join_kernel<E, HD, 1>,
                     dim3((unsigned)(blocks * p.n_seqs)), dim3(256), (size_t)0, st, true, p, (int)blocks));
  }
  return 0;
}

// `rows` of each page; those past it read as zeros.
bool page_map(CUtensorMap* m, const laya_kv_pages& c, const void* base, int rows = 64) {
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)rows, (uint64_t)c.kv_heads, (uint64_t)c.pages};
  const uint64_t strides[3] = {(uint64_t)c.row_stride * 2, (uint64_t)c.head_stride * 2, (uint64_t)c.page_stride * 2};
  const uint32_t box[4] = {64, 64, 1, 1};
  return encode_tiled(m, c.type == LAYA_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

}  // namespace laya

using namespace laya;

extern "C" size_t laya_prefix_attention_workspace(const laya_kv_pages* cache, const laya_prefix_args* a) {
  size_t n = 0;
  guarded([&]() -> int {
    if (int rc = check_sizes(cache, a)) return rc;
    DeviceInfo di;
    if (int rc = device_info(&di)) return rc;
    n = workspace_of(*cache, *a, shape_of(*cache, *a, di.sms));
    return 0;
  });
  return n;
}

extern "C" int laya_prefix_attention(const laya_kv_pages* cache, const laya_prefix_args* a, void* stream) {
  return guarded([&]() -> int {
    if (int rc = check_sizes(cache, a)) return rc;
    if (!(a->scale > 0.f) || !std::isfinite(a->scale * 1.4426950408889634f))
      return fail(LAYA_E_INVALID, "scale must be positive and finite");
    if (a->rows == 0 || a->n_seqs == 0 || a->max_q == 0) return 0;
    if (!cache->k || !cache->v || !a->q || !a->out || !a->offsets || !a->lens || (a->prefix_len && !a->prefix_pages) ||
        (a->width && !a->tables))
      return fail(LAYA_E_INVALID, "null argument");
    if ((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v) |
         reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15)
      return fail(LAYA_E_INVALID, "q, out and the K/V pages must be 16-byte aligned");
    const int64_t width = (int64_t)a->heads * cache->head_dim;
    if (a->q_stride % 8 || a->out_stride % 8 || a->q_stride < 0 ||
        (a->rows > 1 && (a->q_stride < width || a->out_stride < width)))
      return fail(LAYA_E_INVALID, "query and output rows must not overlap and start on 16 bytes");
    if (a->table_stride < a->width) return fail(LAYA_E_INVALID, "block table rows overlap");
    DeviceInfo di;
    if (int rc = device_info(&di)) return rc;
    const Shape s = shape_of(*cache, *a, di.sms);
    const size_t need = workspace_of(*cache, *a, s);
    if (need && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 255)))
      return fail(LAYA_E_INVALID, "workspace missing, misaligned or smaller than laya_prefix_attention_workspace");
    PfxParams p{};
    p.q = a->q;
    p.q_stride = a->q_stride;
    p.rows = a->rows;
    p.H = a->heads;
    p.KV = cache->kv_heads;
    p.G = a->heads / cache->kv_heads;
    p.offsets = a->offsets;
    p.n_seqs = a->n_seqs;
    p.max_q = a->max_q;
    p.prefix_pages = a->prefix_pages;
    p.prefix_len = a->prefix_len;
    p.tables = a->tables;
    p.tstride = a->table_stride;
    p.width = a->width;
    p.lens = a->lens;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.out = a->out;
    p.out_stride = a->out_stride;
    p.lse = a->lse;
    p.sp = s.sp;
    p.ss = s.ss;
    const size_t planes = s.sp || s.ss > 1 ? s.sp + s.ss : 0;
    p.part_l = static_cast<float*>(a->workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(a->workspace) +
                                        align256(planes * (size_t)a->rows * a->heads * 4));
    p.pages = cache->pages;
    p.status = di.status;
    CUtensorMap tq{}, tk, tv, tv_last{};
    bool ok = page_map(&tk, *cache, cache->k) && page_map(&tv, *cache, cache->v);
    if (s.sp && s.tc) {
      p.chunk = s.chunk;
      p.steps = s.steps;
      p.unit_tok = s.unit_tok;
      p.n_units = s.n_units;
      const uint64_t dims[3] = {(uint64_t)cache->head_dim, (uint64_t)a->heads, (uint64_t)a->rows};
      const uint64_t strides[2] = {(uint64_t)cache->head_dim * 2, (uint64_t)a->q_stride * 2};
      const uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)(128 / p.G)};
      ok = ok && page_map(&tv_last, *cache, cache->v, (a->prefix_len - 1) % 64 + 1) &&
           encode_tiled(&tq,
                        cache->type == LAYA_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        3, a->q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (!ok) return fail(LAYA_E_INVALID, "queries or K/V pages that no tensor map can describe");
    auto st = static_cast<cudaStream_t>(stream);
    const bool f16 = cache->type == LAYA_TYPE_F16;
#define LAYA_PFX(HD)                                                                          \
  if (cache->head_dim == HD)                                                                  \
    return f16 ? prefix_go<half, HD>(tq, tk, tv, tv_last, p, s, di.device, di.sms, st)        \
               : prefix_go<__nv_bfloat16, HD>(tq, tk, tv, tv_last, p, s, di.device, di.sms, st);
    LAYA_PFX(64)
    LAYA_PFX(128)
    LAYA_PFX(256)
#undef LAYA_PFX
    return fail(LAYA_E_INVALID, "unsupported head_dim");
  });
}
