// Page plans and K/V append for caller-owned pages, and the status word of
// the device operators.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "device_ops.h"

namespace laya {

__device__ unsigned g_device_status, g_status_taken;

// Reads and clears the status word in one step: a kernel that sets a bit
// meanwhile, on any stream, has it in this reading or the next.
__global__ void take_status_kernel() { g_status_taken = atomicExch(&g_device_status, 0u); }

int device_info(DeviceInfo* out) {
  constexpr int kMax = 64;
  static std::mutex mu;
  static DeviceInfo known[kMax];
  int dev = 0;
  LAYA_CK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMax) return fail(LAYA_E_INVALID, "device index out of range");
  std::lock_guard<std::mutex> lk(mu);
  if (!known[dev].status) {
    int major = 0, sms = 0;
    LAYA_CK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    LAYA_CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (major != 10) return fail(LAYA_E_CUDA, "not an sm_100 GPU");
    void* p = nullptr;
    LAYA_CK(cudaGetSymbolAddress(&p, g_device_status));
    known[dev] = {dev, sms, static_cast<unsigned*>(p)};
  }
  *out = known[dev];
  return 0;
}

int check_pages(const laya_kv_pages* c) {
  if (!c) return fail(LAYA_E_INVALID, "null cache");
  if (c->type != LAYA_TYPE_F16 && c->type != LAYA_TYPE_BF16) return fail(LAYA_E_INVALID, "K/V pages must be F16 or BF16");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(LAYA_E_INVALID, "head_dim must be 64, 128 or 256");
  if (c->pages < 1 || c->kv_heads < 1) return fail(LAYA_E_INVALID, "empty K/V cache");
  const int64_t most = (int64_t)1 << 38;  // a stride's bytes stay below 2^40, the tensor maps' limit
  for (int64_t s : {c->page_stride, c->head_stride, c->row_stride})
    if (s < 0 || s % 8 || s >= most) return fail(LAYA_E_INVALID, "K/V page strides must be multiples of 8 elements");
  return 0;
}

// ------------------------------------------------------------ page plan
//
// have = ceil(past / 64), fresh = ceil((past + count) / 64) - have (cut at
// the table's width); the exclusive prefix sums of count and fresh give a
// sequence's first row and first free page.  Bound by latency for a decode
// step and by the 16 bytes written per token row for prompts.  Every CTA
// computes the prefix sums of all sequences itself (n <= 8192: at most 64 KB
// from L2 into shared memory), so one launch serves both and no CTA waits for
// another; then the CTAs share the table rows and the token rows, each
// thread finding its rows' sequence by a binary search in shared memory.

__device__ __forceinline__ int plan_fresh(int past, int count, int width) {
  const long long have = ((long long)past + 63) / 64, need = ((long long)past + count + 63) / 64;
  return (int)max(0ll, min(need, (long long)width) - have);
}

template <int kPlanThreads>
__global__ void __launch_bounds__(kPlanThreads)
    page_plan_kernel(const int* __restrict__ past, const int* __restrict__ count, int n,
                     const int* __restrict__ free_pages, int n_free, int base, int* __restrict__ tables,
                     long long tstride, int width, long long* __restrict__ slots, int* __restrict__ positions,
                     int* __restrict__ seqs, int capacity, int* __restrict__ offsets, int* __restrict__ lens,
                     long long* __restrict__ totals) {
  extern __shared__ int plan_sm[];
  int* off = plan_sm;          // [n + 1] first rows, cut at the capacity
  int* pg = off + n + 1;       // [n] first free page, cut at n_free
  int* pst = pg + n;           // [n] past
  __shared__ long long wsum[2][kPlanThreads / 32 + 1];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  // sizes into shared memory, coalesced and four loads at a time
#pragma unroll 4
  for (int i = tid; i < n; i += kPlanThreads) {
    pst[i] = max(past[i], 0);
    off[i] = max(count[i], 0);
  }
  __syncthreads();
  // runs of an odd number of sequences per thread: no bank is met twice
  const int per = (n + kPlanThreads - 1) / kPlanThreads | 1;
  const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
  long long st = 0, sp = 0;
  for (int i = i0; i < i1; i++) {
    const int f = plan_fresh(pst[i], off[i], width);
    pg[i] = f;
    st += off[i];
    sp += f;
  }
  long long et = st, ep = sp;  // inclusive over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, et, o), b = __shfl_up_sync(0xffffffffu, ep, o);
    if (lane >= o) {
      et += a;
      ep += b;
    }
  }
  if (lane == 31) {
    wsum[0][warp] = et;
    wsum[1][warp] = ep;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive sums of the warps, and the totals behind them
    const long long t0 = lane < kPlanThreads / 32 ? wsum[0][lane] : 0, p0 = lane < kPlanThreads / 32 ? wsum[1][lane] : 0;
    long long t = t0, q = p0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, t, o), y = __shfl_up_sync(0xffffffffu, q, o);
      if (lane >= o) {
        t += x;
        q += y;
      }
    }
    if (lane < kPlanThreads / 32) {
      wsum[0][lane] = t - t0;
      wsum[1][lane] = q - p0;
    }
    if (lane == 31) {
      wsum[0][kPlanThreads / 32] = t;
      wsum[1][kPlanThreads / 32] = q;
    }
  }
  __syncthreads();
  long long bt = et - st + wsum[0][warp], bp = ep - sp + wsum[1][warp];
  const long long all_t = wsum[0][kPlanThreads / 32], all_p = wsum[1][kPlanThreads / 32];
  for (int i = i0; i < i1; i++) {
    const int c = off[i], f = pg[i];
    off[i] = (int)min(bt, (long long)capacity);
    pg[i] = (int)min(bp, (long long)n_free);
    bt += c;
    bp += f;
  }
  if (tid == 0) off[n] = (int)min(all_t, (long long)capacity);
  __syncthreads();
  // table rows, lengths and offsets: a warp per sequence
  for (int i = blockIdx.x * (kPlanThreads / 32) + warp; i < n; i += gridDim.x * (kPlanThreads / 32)) {
    const int p = pst[i], c = max(count[i], 0);
    const int f = plan_fresh(p, c, width), have = (int)(((long long)p + 63) / 64);
    int* row = tables + (long long)i * tstride;
    for (int a = lane; a < f; a += 32) row[have + a] = a < n_free - pg[i] ? free_pages[pg[i] + a] : -1;
    if (lane == 0) {
      offsets[i] = off[i];
      lens[i] = (int)min((long long)p + c, 2147483647ll);
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    offsets[n] = off[n];
    totals[0] = all_t;
    totals[1] = all_p;
  }
  // token rows, four at a time per thread
  const int total = off[n];
  const long long step = (long long)gridDim.x * kPlanThreads * 4;
  for (long long t0 = ((long long)blockIdx.x * kPlanThreads + tid) * 4; t0 < capacity; t0 += step) {
    int i = n;
    if (t0 < total) {  // the last sequence with off[i] <= t0
      int lo = 0, hi = n;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (off[mid] <= t0)
          lo = mid;
        else
          hi = mid;
      }
      i = lo;
    }
    // places fit 32 unsigned bits: past and count are below 2^31
    long long sl[4];
    int po[4], se[4];
    unsigned known = 0xffffffffu;  // page index that `page` is of
    int page = -1;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const long long t = t0 + e;
      sl[e] = -1;
      po[e] = 0;
      se[e] = -1;
      if (t < total) {
        if (off[i + 1] <= t) {
          while (off[i + 1] <= t) i++;  // ends: off[n] = total > t
          known = 0xffffffffu;
        }
        const unsigned u = (unsigned)pst[i] + (unsigned)((int)t - off[i]), b = u / 64;
        if (b != known) {
          const unsigned have = ((unsigned)pst[i] + 63u) / 64;
          known = b;
          page = -1;
          if (b < (unsigned)width) {
            if (b < have)
              page = tables[(long long)i * tstride + b];
            else if (b - have < (unsigned)(n_free - pg[i]))
              page = free_pages[pg[i] + (int)(b - have)];
          }
        }
        if (page >= 0) sl[e] = (long long)page * 64 + (u & 63);
        po[e] = (int)((unsigned)base + u);
        se[e] = i;
      }
    }
    if (t0 + 4 <= capacity) {
      reinterpret_cast<longlong2*>(slots + t0)[0] = make_longlong2(sl[0], sl[1]);
      reinterpret_cast<longlong2*>(slots + t0)[1] = make_longlong2(sl[2], sl[3]);
      if (positions) *reinterpret_cast<int4*>(positions + t0) = make_int4(po[0], po[1], po[2], po[3]);
      if (seqs) *reinterpret_cast<int4*>(seqs + t0) = make_int4(se[0], se[1], se[2], se[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (t0 + e < capacity) {
          slots[t0 + e] = sl[e];
          if (positions) positions[t0 + e] = po[e];
          if (seqs) seqs[t0 + e] = se[e];
        }
    }
  }
}

// ------------------------------------------------------------ K/V append
//
// A copy of rows into scattered slots, bound by HBM: 2 rows x kv_heads x
// head_dim read and written once.  A warp takes one row of K or of V; lane l
// moves 16-byte pieces l, l + 32, ... of it, four loads in flight per lane.
template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<half>(float a, float b) {
  half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename E, bool F32>
__global__ void __launch_bounds__(256)
    kv_append_kernel(laya_kv_pages c, const void* __restrict__ k, const void* __restrict__ v, long long ks,
                     long long vs, const long long* __restrict__ slots, int rows, int log_hd8, unsigned* status) {
  const int lane = threadIdx.x % 32;
  const int pieces = c.kv_heads << log_hd8;
  const long long n_slots = (long long)c.pages * 64;
  const long long warps = (long long)gridDim.x * 8;
  for (long long w = (long long)blockIdx.x * 8 + threadIdx.x / 32; w < 2ll * rows; w += warps) {
    const long long t = w >> 1;
    const bool is_v = w & 1;
    const long long slot = slots[t];
    if (slot < 0 || slot >= n_slots) {
      if (slot != -1 && lane == 0) atomicOr(status, LAYA_STATUS_PAGE);
      continue;
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<E*>(is_v ? c.v : c.k) + (slot >> 6) * c.page_stride +
                                          (slot & 63) * c.row_stride);
    const long long hs = c.head_stride / 8;
    const long long first = t * (is_v ? vs : ks);
    for (int p0 = lane; p0 < pieces; p0 += 128) {
      uint4 x[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int p = p0 + 32 * e;
        if (p >= pieces) continue;
        if constexpr (F32) {
          const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(is_v ? v : k) + first) + 2 * p;
          const float4 a = __ldg(s), b = __ldg(s + 1);
          x[e] = make_uint4(pack2<E>(a.x, a.y), pack2<E>(a.z, a.w), pack2<E>(b.x, b.y), pack2<E>(b.z, b.w));
        } else {
          x[e] = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(is_v ? v : k) + first) + p);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int p = p0 + 32 * e;
        if (p < pieces) dst[(p >> log_hd8) * hs + (p & ((1 << log_hd8) - 1))] = x[e];
      }
    }
  }
}

}  // namespace laya

using namespace laya;

extern "C" int laya_device_status(int device, uint32_t* bits) {
  return guarded([&]() -> int {
    if (!bits) return fail(LAYA_E_INVALID, "null argument");
    int before = 0;
    LAYA_CK(cudaGetDevice(&before));
    LAYA_CK(cudaSetDevice(device));
    static std::mutex mu;  // g_status_taken is one call's at a time
    std::lock_guard<std::mutex> lk(mu);
    DeviceInfo di;
    int rc = device_info(&di);
    unsigned got = 0;
    cudaError_t e = cudaSuccess;
    if (!rc) {
      e = cudaDeviceSynchronize();
      if (e == cudaSuccess) {
        take_status_kernel<<<1, 1>>>();
        e = cudaGetLastError();
      }
      if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&got, g_status_taken, 4);
    }
    cudaSetDevice(before);
    if (rc) return rc;
    if (e != cudaSuccess) return cuda_fail(e, "laya_device_status");
    *bits = got;
    return 0;
  });
}

extern "C" int laya_page_plan(const int32_t* past, const int32_t* count, int n, const int32_t* free_pages, int n_free,
                              int base, int32_t* tables, int64_t table_stride, int width, int64_t* slots,
                              int32_t* positions, int32_t* seqs, int capacity, int32_t* offsets, int32_t* lens,
                              int64_t* totals, void* stream) {
  return guarded([&]() -> int {
    if (n < 0 || n_free < 0 || width < 0 || capacity < 0 || table_stride < width)
      return fail(LAYA_E_INVALID, "negative size in page plan, or table rows that overlap");
    if (n > LAYA_PLAN_MAX_SEQS) return fail(LAYA_E_INVALID, "a page plan holds at most 8192 sequences");
    if ((n && (!past || !count || !lens)) || (n && width && !tables) || (n_free && !free_pages) ||
        (capacity && !slots) || !offsets || !totals)
      return fail(LAYA_E_INVALID, "null argument");
    if ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions) |
         reinterpret_cast<uintptr_t>(seqs)) & 15)
      return fail(LAYA_E_INVALID, "slots, positions and seqs must be 16-byte aligned");
    DeviceInfo di;
    if (int rc = device_info(&di)) return rc;
    const size_t smem = ((size_t)3 * n + 1) * 4;
    static std::atomic<bool> configured[64];
    if (!configured[di.device & 63]) {
      LAYA_CK(cudaFuncSetAttribute(page_plan_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (3 * LAYA_PLAN_MAX_SEQS + 1) * 4));
      configured[di.device & 63] = true;
    }
    auto go = [&](auto kernel, int threads, int grid) {
      kernel<<<grid, threads, smem, static_cast<cudaStream_t>(stream)>>>(
          past, count, n, free_pages, n_free, base, tables, table_stride, width, reinterpret_cast<long long*>(slots),
          positions, seqs, capacity, offsets, lens, reinterpret_cast<long long*>(totals));
    };
    // A decode step is one small CTA or a few; otherwise one CTA per 4096 token
    // rows or 32 sequences and at most one per SM: more would only repeat the
    // prefix sums (4096 sequences, 1 M rows, before the sums and lookups got
    // shorter: 14.4 us; two per SM 14.7, four 19.2; the present code 11.3).
    const int64_t want = std::max<int64_t>((capacity + 4095ll) / 4096, (n + 31) / 32);
    if (n <= 1024 && capacity <= 8192)
      go(page_plan_kernel<256>, 256, (int)std::max<int64_t>(1, std::max<int64_t>((capacity + 1023ll) / 1024, (n + 63) / 64)));
    else
      go(page_plan_kernel<1024>, 1024, (int)std::min<int64_t>(want, di.sms));
    LAYA_CK(cudaGetLastError());
    return 0;
  });
}

extern "C" int laya_kv_append(const laya_kv_pages* cache, uint32_t type, const void* k, const void* v,
                              int64_t k_stride, int64_t v_stride, const int64_t* slots, int rows, void* stream) {
  return guarded([&]() -> int {
    if (int rc = check_pages(cache)) return rc;
    if (type != cache->type && type != LAYA_TYPE_F32)
      return fail(LAYA_E_INVALID, "K/V rows must be of the cache's type or F32");
    if (rows < 0) return fail(LAYA_E_INVALID, "negative row count");
    if (rows == 0) return 0;
    if (!cache->k || !cache->v || !k || !v || !slots) return fail(LAYA_E_INVALID, "null argument");
    const int64_t unit = type == LAYA_TYPE_F32 ? 4 : 8, width = (int64_t)cache->kv_heads * cache->head_dim;
    if (k_stride % unit || v_stride % unit || k_stride < 0 || v_stride < 0 ||
        ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(cache->k) |
          reinterpret_cast<uintptr_t>(cache->v)) & 15))
      return fail(LAYA_E_INVALID, "K/V rows and pages must be 16-byte aligned");
    if (rows > 1 && (k_stride < width || v_stride < width)) return fail(LAYA_E_INVALID, "K/V rows overlap");
    if (width > (1 << 24)) return fail(LAYA_E_INVALID, "K/V rows too wide");
    DeviceInfo di;
    if (int rc = device_info(&di)) return rc;
    const int log_hd8 = cache->head_dim == 64 ? 3 : cache->head_dim == 128 ? 4 : 5;
    const int grid = (int)std::min<int64_t>((2ll * rows + 7) / 8, 16ll * di.sms);
    auto st = static_cast<cudaStream_t>(stream);
    auto s64 = reinterpret_cast<const long long*>(slots);
#define LAYA_APPEND(E, F32)                                                                                       \
  kv_append_kernel<E, F32><<<grid, 256, 0, st>>>(*cache, k, v, k_stride, v_stride, s64, rows, log_hd8, di.status)
    if (cache->type == LAYA_TYPE_F16) {
      if (type == LAYA_TYPE_F32) LAYA_APPEND(half, true); else LAYA_APPEND(half, false);
    } else {
      if (type == LAYA_TYPE_F32) LAYA_APPEND(__nv_bfloat16, true); else LAYA_APPEND(__nv_bfloat16, false);
    }
#undef LAYA_APPEND
    LAYA_CK(cudaGetLastError());
    return 0;
  });
}
