// tkv_kv8.cu -- step planning, rotary positions and the quantizing append of
// the 8-bit paged cache (tkv_kv8_* in include/tierkv_b200.h).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tierkv_b200.h"
#include "tkv_kv8.h"
#include "tkv_ptx.cuh"

namespace cg = cooperative_groups;

namespace tkv {

// ---------------------------------------------------------------- step planning
//
// need(i) = ceil((c + n) / bs) - ceil(c / bs) new blocks, C their running sum;
// the k-th block of the step is the k-th from the end of the free list.  One
// cluster plans the step: every CTA scans the requests' lengths into shared
// memory (an 8-byte load per request, so repeating it per CTA costs nothing
// next to a second launch), then the cluster's threads share the tokens, table
// cells and write units and find each one's request by bisection of the
// scanned sums.  A cluster barrier between the last read of an input and the
// first write lets kv_lens / free_count be updated in place.  Latency bound:
// a launch, one round of loads, two block scans (64 requests of one token: 4.5
// us; 1024 requests with 130000 tokens: 10.1 us for 1.7 MB of outputs).
// Small steps (up to 1024 requests, tokens and write units) take one CTA of 256
// threads, whose barriers are cheaper than the cluster's; others 16 of 1024, the
// largest cluster there is (8: 13.3 us for those 130000 tokens, 16 of 512: 10.8;
// 2000 tokens the same), or 8, which every device can place, where a part of a
// GPU has no room for 16.
#ifndef TKV_PLAN_CLUSTER
#define TKV_PLAN_CLUSTER 16
#endif
constexpr int kPlanCluster = TKV_PLAN_CLUSTER, kPlanPortable = 8;
constexpr int kPlanThreads = 1024, kPlanSmall = 256;
constexpr int kPlanSmallWork = 1024;

struct Scan {
  int32_t warp_sum[2][32];
  int32_t carry[2];
};

// a + b for a, b >= 0, at most 2^31 - 1: sums over lengths that make no sense
// (8192 prompts of 2^30 tokens) stay sums that no step can hold.
__device__ __forceinline__ int32_t sat_add(int32_t a, int32_t b) {
  return (int32_t)min((uint32_t)a + (uint32_t)b, 0x7fffffffu);
}

// Exclusive saturated sums over the CTA's threads of (a, b); every thread also gets the totals.
__device__ __forceinline__ void scan2(Scan& s, int32_t a, int32_t b, int32_t& ea, int32_t& eb,
                                      int32_t& ta, int32_t& tb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t xa = __shfl_up_sync(~0u, ia, o), xb = __shfl_up_sync(~0u, ib, o);
    if (lane >= o) {
      ia = sat_add(ia, xa);
      ib = sat_add(ib, xb);
    }
  }
  __syncthreads();  // the previous scan's readers are done
  if (lane == 31) {
    s.warp_sum[0][warp] = ia;
    s.warp_sum[1][warp] = ib;
  }
  __syncthreads();
  const bool has = lane < (int)blockDim.x / 32;
  int32_t wa = has ? s.warp_sum[0][lane] : 0, wb = has ? s.warp_sum[1][lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t xa = __shfl_up_sync(~0u, wa, o), xb = __shfl_up_sync(~0u, wb, o);
    if (lane >= o) {
      wa = sat_add(wa, xa);
      wb = sat_add(wb, xb);
    }
  }
  ta = __shfl_sync(~0u, wa, 31);
  tb = __shfl_sync(~0u, wb, 31);
  const int32_t before_a = __shfl_sync(~0u, wa, warp ? warp - 1 : 0);
  const int32_t before_b = __shfl_sync(~0u, wb, warp ? warp - 1 : 0);
  const int32_t lane_a = __shfl_up_sync(~0u, ia, 1), lane_b = __shfl_up_sync(~0u, ib, 1);
  ea = sat_add(warp ? before_a : 0, lane ? lane_a : 0);
  eb = sat_add(warp ? before_b : 0, lane ? lane_b : 0);
}

// Largest i with first[i] <= x, for a non-decreasing first[0 .. n] with first[0] = 0 <= x < first[n].
__device__ __forceinline__ int find(const int32_t* first, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// x / 2^log2, rounded up, for any x below 2^32.
__device__ __forceinline__ int32_t ceil_div(uint32_t x, int log2) {
  return (int32_t)((x >> log2) + ((x & ((1u << log2) - 1)) != 0));
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1)
    plan_step_kernel(const __grid_constant__ tkv_kv8_plan_args p) {
  extern __shared__ int32_t plan_smem[];
  __shared__ Scan scan;
  const cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  pdl_wait();
  const int n = p.requests, bs = p.block_size, bs_log2 = 31 - __clz(bs), tid = threadIdx.x;
  int32_t* ctx = plan_smem;            // [n]      cached tokens, bit 31: not admitted
  int32_t* cu = ctx + n;               // [n + 1]  first packed token
  int32_t* need = cu + n + 1;          // [n + 1]  running sum of new blocks
  int32_t* cu_unit = need + n + 1;     // [n + 1]  first write unit
  const int32_t free_count = max(0, min(*p.free_count, p.free_capacity));

  // lengths -> running sums of the new tokens and the new blocks; a thread
  // owns n / kThreads consecutive requests
  const int per = (n + kThreads - 1) / kThreads;
  const int r0 = min(n, tid * per), r1 = min(n, r0 + per);
  int32_t sum_new = 0, sum_need = 0;
  for (int i = r0; i < r1; ++i) {
    const int32_t c = max(0, p.context_lens[i]), m = max(0, p.new_lens[i]);
    const int32_t want = ceil_div((uint32_t)c + (uint32_t)m, bs_log2);
    ctx[i] = c;
    cu[i] = m;
    need[i] = want <= p.table_width ? want - ceil_div(c, bs_log2) : -1;
    sum_new = sat_add(sum_new, m);
    sum_need = sat_add(sum_need, max(0, need[i]));
  }
  int32_t at_new, at_need, total_new, total_need;
  scan2(scan, sum_new, sum_need, at_new, at_need, total_new, total_need);
  int32_t sum_units = 0, taken = 0;
  bool refused = false;
  for (int i = r0; i < r1; ++i) {
    const int32_t m = cu[i], k = need[i], c = ctx[i];
    const bool ok = k >= 0 && (k == 0 || (uint32_t)at_need + (uint32_t)k <= (uint32_t)free_count);
    if (!ok) ctx[i] = c | (int32_t)0x80000000;
    if (!ok && m > 0) refused = true;
    cu[i] = at_new;
    need[i] = at_need;
    cu_unit[i] = ok && m > 0 ? ceil_div(c + m, bs_log2) - (c >> bs_log2) : 0;
    sum_units = sat_add(sum_units, cu_unit[i]);
    at_new = sat_add(at_new, m);
    at_need = sat_add(at_need, max(0, k));
    if (ok) taken += k;                   // free_count at most, in sum
  }
  int32_t at_unit, at_taken, total_units, total_taken;
  scan2(scan, sum_units, taken, at_unit, at_taken, total_units, total_taken);
  for (int i = r0; i < r1; ++i) {
    const int32_t u = cu_unit[i];
    cu_unit[i] = at_unit;
    at_unit = sat_add(at_unit, u);
  }
  if (tid == 0) {
    cu[n] = total_new;
    need[n] = total_need;
    cu_unit[n] = total_units;
  }
  cluster.sync();  // every CTA has read its inputs; shared memory is complete

  const int rank = (int)cluster.block_rank();
  const uint32_t gtid = rank * kThreads + tid;
  const uint32_t stride = cluster.num_blocks() * kThreads;
  const bool vec = ((reinterpret_cast<uintptr_t>(p.slot_map) | reinterpret_cast<uintptr_t>(p.token_request) |
                     reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0;
  if (rank == 0) {
    for (int i = r0; i < r1; ++i) {
      const int32_t c = ctx[i] & 0x7fffffff;
      const int32_t m = cu[i + 1] < 0x7fffffff ? cu[i + 1] - cu[i] : max(0, p.new_lens[i]);
      p.kv_lens[i] = ctx[i] >= 0 ? c + m : c;
      p.cu_q[i] = cu[i];
      p.admitted[i] = ctx[i] >= 0;
    }
    if (tid == 0) {
      p.cu_q[n] = total_new;
      *p.num_units = min(total_units, p.units_cap);
      *p.free_count_out = free_count - total_taken;
    }
    if (refused && p.error_word) atomicOr(p.error_word, TKV_DEVERR_NO_BLOCKS);
    if (tid == 0 && p.tokens > 0 && total_new > p.tokens && p.error_word) atomicOr(p.error_word, TKV_DEVERR_DROPPED);
  }

  // new table cells; blocks past the free list are nobody's
  for (uint32_t u = gtid; u < (uint32_t)min(total_need, free_count); u += stride) {
    const int i = find(need, n, u);
    if (ctx[i] < 0) continue;
    p.block_table[i * p.table_stride + ceil_div(ctx[i], bs_log2) + (u - need[i])] =
        p.free_blocks[free_count - 1 - u];
  }
  // block of request i's cell j: one this step takes, or one it already held
  auto block_of = [&](int i, int32_t c, int32_t j) -> int32_t {
    const int32_t held = ceil_div(c, bs_log2);
    return j >= held ? p.free_blocks[free_count - 1 - (need[i] + j - held)]
                     : p.block_table[i * p.table_stride + j];
  };
  // write units
  for (uint32_t u = gtid; u < (uint32_t)p.units_cap; u += stride) {
    int4 out = make_int4(-1, -1, -1, -1);
    if (u < (uint32_t)total_units) {
      const int i = find(cu_unit, n, u);
      const int32_t c = ctx[i], end = c + (cu[i + 1] - cu[i]);
      const int32_t j = (c >> bs_log2) + (u - cu_unit[i]);
      const int32_t lo = max(c, j * bs), hi = min(end, (j + 1) * bs);
      out = make_int4(block_of(i, c, j), cu[i] + (lo - c), lo - j * bs, hi - lo);
    }
    reinterpret_cast<int4*>(p.units)[u] = out;
  }
  // tokens, four consecutive ones at a time: they share a request or two and
  // mostly a block, and leave as 16-byte stores
  for (uint32_t t0 = 4 * gtid; t0 < (uint32_t)p.tokens; t0 += 4 * stride) {
    int4 slot = make_int4(-1, -1, -1, -1), rq = slot, ps = slot;
    if (t0 < (uint32_t)total_new) {
      int req = find(cu, n, t0), end = cu[req + 1], c = ctx[req], cell = -1, cell_at = -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = (int)t0 + k;
        if (t0 + k >= (uint32_t)total_new) break;
        if (t >= end) {
          do ++req; while (cu[req + 1] <= t);
          end = cu[req + 1];
          c = ctx[req];
          cell_at = -1;
        }
        const int pos = sat_add(c & 0x7fffffff, t - cu[req]);   // a refused request's context is any number
        const int j = pos >> bs_log2;
        if (c >= 0 && j != cell_at) {
          cell = block_of(req, c, j);
          cell_at = j;
        }
        reinterpret_cast<int*>(&slot)[k] = c >= 0 ? (cell << bs_log2) + (pos & (bs - 1)) : -1;
        reinterpret_cast<int*>(&rq)[k] = req;
        reinterpret_cast<int*>(&ps)[k] = pos;
      }
    }
    if (t0 + 4 <= (uint32_t)p.tokens && vec) {
      *reinterpret_cast<int4*>(p.slot_map + t0) = slot;
      *reinterpret_cast<int4*>(p.token_request + t0) = rq;
      *reinterpret_cast<int4*>(p.positions + t0) = ps;
    } else {
      for (int k = 0; k < 4 && t0 + k < (uint32_t)p.tokens; ++k) {
        p.slot_map[t0 + k] = reinterpret_cast<int*>(&slot)[k];
        p.token_request[t0 + k] = reinterpret_cast<int*>(&rq)[k];
        p.positions[t0 + k] = reinterpret_cast<int*>(&ps)[k];
      }
    }
  }
}

// CTAs of the current device's plan cluster, with the kernel's opt-ins made.
static cudaError_t plan_cluster(int* ctas) {
  static std::atomic<int> known[kKv8MaxDevices];
  static std::atomic<uint64_t> allowed, wide;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool cached = dev >= 0 && dev < kKv8MaxDevices;
  if (cached && (*ctas = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  const int smem = (int)(sizeof(int32_t) * (4 * TKV_KV8_MAX_REQUESTS + 3));
  if ((e = allow_smem(plan_step_kernel<kPlanThreads>, smem, allowed)) != cudaSuccess) return e;
  *ctas = kPlanPortable;
  if (allow(plan_step_kernel<kPlanThreads>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1, wide) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kPlanCluster);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPlanCluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, plan_step_kernel<kPlanThreads>, &cfg) == cudaSuccess && fit > 0)
      *ctas = kPlanCluster;
  }
  cudaGetLastError();   // a size that does not fit is no error of this call
  if (cached) known[dev].store(*ctas, std::memory_order_relaxed);
  return cudaSuccess;
}

cudaError_t launch_plan_step(const tkv_kv8_plan_args& p, cudaStream_t stream) {
  const size_t smem = sizeof(int32_t) * (4 * (size_t)p.requests + 3);
  const bool small = p.requests <= kPlanSmallWork && p.tokens <= kPlanSmallWork && p.units_cap <= kPlanSmallWork;
  int ctas = 1;
  if (!small) {
    const cudaError_t e = plan_cluster(&ctas);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(small ? kPlanSmall : kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cfg.gridDim.x;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = small ? 1 : 2;
  return small ? cudaLaunchKernelEx(&cfg, plan_step_kernel<kPlanSmall>, p)
               : cudaLaunchKernelEx(&cfg, plan_step_kernel<kPlanThreads>, p);
}

// ---------------------------------------------------------------- element types
template <typename T>
struct Pack;  // 8 elements in 16 bytes
template <>
struct Pack<__half> {
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    return v;
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    return v;
  }
};

// ---------------------------------------------------------------- rotation
// A rotation item is 16 elements of one head: 8 frequencies f0 .. f0 + 7 and
// both elements of their pairs, held as x[0..7] (x1) and x[8..15] (x2).  Items
// past rot_dim / 16 are 16 consecutive elements that pass through.
struct ItemPlace {
  int lo, hi;  // element offsets of the item's two 16-byte halves
  int f0;      // first frequency, -1: passes through
};
__device__ __forceinline__ ItemPlace item_place(const RotaryArgs& r, int item) {
  ItemPlace w;
  if (item < r.rot_dim / 16) {
    w.f0 = item * 8;
    w.lo = r.pairs ? item * 16 : item * 8;
    w.hi = r.pairs ? item * 16 + 8 : r.rot_dim / 2 + item * 8;
  } else {
    w.f0 = -1;
    w.lo = item * 16;
    w.hi = w.lo + 8;
  }
  return w;
}

// Axis of frequency f.
__device__ __forceinline__ int freq_axis(const RotaryArgs& r, int f) {
  if (r.axes == 1) return 0;
  if (r.interleave) {
    const int a = f % r.axes;
    return f / r.axes < r.sections[a] ? a : 0;
  }
  int a = 0, end = r.sections[0];
  while (f >= end && a + 1 < r.axes) end += r.sections[++a];
  return a;
}

__device__ __forceinline__ int64_t load_position(const RotaryArgs& r, int axis, int64_t token,
                                                 uint32_t* err) {
  const int64_t at = axis * r.axis_stride + token;
  const int64_t p = r.positions_bytes == 8 ? reinterpret_cast<const int64_t*>(r.positions)[at]
                                           : (int64_t)reinterpret_cast<const int32_t*>(r.positions)[at];
  if (p >= 0 && p < r.rows) return p;
  if (p != -1 && err) atomicOr(err, TKV_DEVERR_BAD_POS);   // -1: a step's padding
  return p < 0 ? 0 : r.rows - 1;
}

// y1 = x1 c - x2 s, y2 = x2 c + x1 s; every product and sum rounded by itself,
// so that codes quantized from the result equal an unfused pipeline's.
__device__ __forceinline__ void turn(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
}

// The pair order of `pairs` (x1, x2 adjacent) <-> the split order (all x1, all x2).
__device__ __forceinline__ void split_pairs(float (&x)[16]) {
  float y[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = x[2 * i];
    y[8 + i] = x[2 * i + 1];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = y[i];
}
__device__ __forceinline__ void join_pairs(float (&x)[16]) {
  float y[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[2 * i] = x[i];
    y[2 * i + 1] = x[8 + i];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = y[i];
}

template <typename T>
__device__ __forceinline__ void load_item(const T* row, const ItemPlace& w, float (&x)[16]) {
  float a[8], b[8];
  Pack<T>::unpack(*reinterpret_cast<const uint4*>(row + w.lo), a);
  Pack<T>::unpack(*reinterpret_cast<const uint4*>(row + w.hi), b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = a[i];
    x[8 + i] = b[i];
  }
}

// One CTA rotates every head of one token: (c, s) of its rot_dim / 2
// frequencies go to shared memory once (the table row is 4 rot_dim bytes
// against 2 head_dim bytes of each head), then the threads share the (head,
// item) pairs.  Bound by HBM: every element is read once and written once
// (16385 tokens of 40 heads of 128, bf16, three axes: 67 us, 5.1 TB/s).
constexpr int kRotThreads = 128;
constexpr int kMaxRotDim = 256;

template <typename T>
__device__ __forceinline__ void rotate_token(const RotaryArgs& r, int64_t token, const T* q, const T* k,
                                             T* qo, T* ko, int64_t qs, int64_t ks, int64_t qos,
                                             int64_t kos, int heads, int kv_heads, int head_dim,
                                             float* cs, uint32_t* err) {
  const int half = r.rot_dim / 2;
  for (int f = threadIdx.x; f < half; f += kRotThreads) {
    const int64_t p = load_position(r, freq_axis(r, f), token, err);
    cs[f] = r.cos_sin[p * r.rot_dim + f];
    cs[half + f] = r.cos_sin[p * r.rot_dim + half + f];
  }
  __syncthreads();
  const int per = head_dim / 16;
  const int total = (heads + kv_heads) * per;
  for (int i = threadIdx.x; i < total; i += kRotThreads) {
    const int h = i / per;
    const ItemPlace w = item_place(r, i - h * per);
    const T* src = h < heads ? q + h * qs : k + (h - heads) * ks;
    T* dst = h < heads ? qo + h * qos : ko + (h - heads) * kos;
    float x[16];
    load_item<T>(src, w, x);
    if (w.f0 >= 0) {
      if (r.pairs) split_pairs(x);
#pragma unroll
      for (int j = 0; j < 8; ++j) turn(x[j], x[8 + j], cs[w.f0 + j], cs[half + w.f0 + j]);
      if (r.pairs) join_pairs(x);
    }
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = x[j];
      b[j] = x[8 + j];
    }
    *reinterpret_cast<uint4*>(dst + w.lo) = Pack<T>::pack(a);
    *reinterpret_cast<uint4*>(dst + w.hi) = Pack<T>::pack(b);
  }
}

template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float cs[kMaxRotDim];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  rotate_token<T>(p.rot, t, (const T*)p.q.data + t * p.q.token_stride,
                  (const T*)p.k.data + t * p.k.token_stride,
                  (T*)const_cast<void*>(p.q_out.data) + t * p.q_out.token_stride,
                  (T*)const_cast<void*>(p.k_out.data) + t * p.k_out.token_stride, p.q.head_stride,
                  p.k.head_stride, p.q_out.head_stride, p.k_out.head_stride, p.heads, p.kv_heads,
                  p.head_dim, cs, p.err);
}

cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream) {
  if (p.tokens == 0 || p.heads + p.kv_heads == 0) return cudaSuccess;
  return launch_dependent(dtype == kDtF16 ? rotary_kernel<__half> : rotary_kernel<__nv_bfloat16>, dim3(p.tokens),
                          kRotThreads, 0, stream, p);
}

// ---------------------------------------------------------------- append
// Quantization to a code byte, to the nearest (ties to even), saturating.
template <int FMT>
__device__ __forceinline__ uint32_t encode(float x) {
  if (FMT == TKV_KV8_INT8) {
    const float q = fminf(fmaxf(rintf(x), -127.f), 127.f);
    return (uint32_t)(int32_t)q & 0xffu;
  }
  return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
template <int FMT>
__device__ __forceinline__ float decode(uint32_t b) {
  if (FMT == TKV_KV8_INT8) return (float)(int8_t)b;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}
template <int FMT>
constexpr float kQMax = FMT == TKV_KV8_INT8 ? 127.f : 448.f;

// Codes of x / s.  x (1 / s) is within 2^-22 of the quotient, so the codes of the
// two ends of that interval agree unless the quotient lies next to a rounding
// boundary; only then (about once in 10^4 elements) it is divided.
template <int FMT>
__device__ __forceinline__ uint32_t encode_quotient(float x, float s, float inv) {
  const float q = x * inv;
  if (!(inv < INFINITY)) return encode<FMT>(__fdiv_rn(x, s));   // 1 / s overflows for a subnormal s
  if (FMT == TKV_KV8_INT8) {
    const float n = rintf(q);
    if (fabsf(fabsf(q - n) - 0.5f) > 1e-4f) return (uint32_t)(int32_t)fminf(fmaxf(n, -127.f), 127.f) & 0xffu;
    return encode<FMT>(__fdiv_rn(x, s));
  }
  const uint32_t a = encode<FMT>(q * (1.f - 0x1p-21f)), b = encode<FMT>(q * (1.f + 0x1p-21f));
  return a == b ? a : encode<FMT>(__fdiv_rn(x, s));
}

template <int FMT>
__device__ __forceinline__ uint2 encode8(const float* x, float s, float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= encode_quotient<FMT>(x[i], s, inv) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

// A tile is one (write unit, K or V, kv head): BS rows of D codes and one
// scale, owned by WPT warps.  Thread layout: D / 16 rotation items per row;
// a warp covers 32 / (D / 16) rows at once.  The tile is walked twice, for its
// maximum and for its codes; the second read of the new rows (at most 16 KB a
// CTA) hits the caches.  Keeping them in registers instead unrolls the walk: the
// instruction fetch and an occupancy of 5 CTAs held it at 63 us for 6000 tokens
// against 51-55 (1.9 TB/s of DRAM; 44 us where the item's frequencies share an
// axis).  Bound by instruction issue, 61 % of the slots.  Old rows are touched only when the scale grows.
template <int D, int BS>
struct AppendShape {
  static constexpr int kPerRow = D / 16;
  static constexpr int kTileItems = BS * kPerRow;
  static constexpr int kWarps = kTileItems / 32 >= 16 ? 4 : (kTileItems / 32 >= 8 ? 2 : 1);
  static constexpr int kItems = kTileItems / (32 * kWarps);
  static constexpr int kTiles = 4 / kWarps;  // per CTA of 128 threads
};

template <typename T, int D, int BS, int FMT>
__global__ void __launch_bounds__(128, 8) append_kernel8(const __grid_constant__ AppendParams8 p) {
  using S = AppendShape<D, BS>;
  __shared__ float cs[kMaxRotDim];
  __shared__ float warp_max[4];
  pdl_launch_dependents();
  pdl_wait();
  const int tiles_per_unit = 2 * p.kv_heads;
  const int ctas_per_unit = (tiles_per_unit + S::kTiles - 1) / S::kTiles;
  const int64_t unit_ctas = (int64_t)p.units_cap * ctas_per_unit;
  if ((int64_t)blockIdx.x >= unit_ctas) {
    // ---- the query's rotation, one token a CTA
    const int64_t t = (int64_t)blockIdx.x - unit_ctas;
    rotate_token<T>(p.rot, t, (const T*)p.q.data + t * p.q.token_stride, (const T*)nullptr,
                    (T*)const_cast<void*>(p.q_out.data) + t * p.q_out.token_stride, (T*)nullptr,
                    p.q.head_stride, 0, p.q_out.head_stride, 0, p.heads, 0, D, cs, p.err);
    return;
  }
  const int u = (int)(blockIdx.x / ctas_per_unit);
  if (u >= min(*p.num_units, p.units_cap)) return;
  const int4 unit = reinterpret_cast<const int4*>(p.units)[u];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = warp / S::kWarps;             // tile of the CTA
  const int part = warp % S::kWarps;            // warp of the tile
  const int tile = (int)(blockIdx.x % ctas_per_unit) * S::kTiles + sub;
  const int off = unit.z, rows = unit.w;
  const bool good = unit.x >= 0 && unit.x < p.blocks && off >= 0 && rows >= 1 && rows <= BS - off &&
                    unit.y >= 0 && unit.y <= p.tokens - rows;
  if (!good) {  // the unit's CTAs agree
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, TKV_DEVERR_BAD_SLOT);
    return;
  }
  const bool live = tile < tiles_per_unit;
  const bool is_v = tile >= p.kv_heads;
  const int h = is_v ? tile - p.kv_heads : tile;
  const int item = lane % S::kPerRow;
  const int row0 = part * (S::kItems * 32 / S::kPerRow) + lane / S::kPerRow;
  constexpr int kRowStep = 32 / S::kPerRow;
  const bool rotate = !is_v && p.has_rot;
  RotaryArgs plain = {};
  const ItemPlace w = item_place(rotate ? p.rot : plain, item);
  const tkv_token_view& view = is_v ? p.v : p.k;
  const T* src = (const T*)view.data + h * view.head_stride;

  // the axes of the item's 8 frequencies, 4 bits each; one for all in most layouts
  uint32_t axes = 0;
  bool one_axis = true;
  if (rotate && w.f0 >= 0 && p.rot.axes > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) axes |= (uint32_t)freq_axis(p.rot, w.f0 + j) << (4 * j);
    one_axis = axes == (axes & 15u) * 0x11111111u;
  }
  // the item of a new row, rotated
  auto fetch = [&](int row, float (&x)[16]) {
    const int64_t token = unit.y + (row - off);
    load_item<T>(src + token * view.token_stride, w, x);
    if (!rotate || w.f0 < 0) return;
    const int half = p.rot.rot_dim / 2;
    if (p.rot.pairs) split_pairs(x);
    if (one_axis) {
      const float* c = p.rot.cos_sin + load_position(p.rot, axes & 15, token, p.err) * p.rot.rot_dim + w.f0;
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(c + j);
        const float4 s4 = *reinterpret_cast<const float4*>(c + half + j);
        turn(x[j], x[8 + j], c4.x, s4.x);
        turn(x[j + 1], x[9 + j], c4.y, s4.y);
        turn(x[j + 2], x[10 + j], c4.z, s4.z);
        turn(x[j + 3], x[11 + j], c4.w, s4.w);
      }
    } else {
      const float* row_of[4];
#pragma unroll
      for (int a = 0; a < 4; ++a)
        row_of[a] = a < p.rot.axes ? p.rot.cos_sin + load_position(p.rot, a, token, p.err) * p.rot.rot_dim + w.f0
                                   : nullptr;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = axes >> (4 * j) & 15;
        const float* c = a == 0 ? row_of[0] : a == 1 ? row_of[1] : a == 2 ? row_of[2] : row_of[3];
        turn(x[j], x[8 + j], c[j], c[half + j]);
      }
    }
    if (p.rot.pairs) join_pairs(x);
  };

  float* scale = (is_v ? p.v_scale : p.k_scale) + (int64_t)unit.x * p.kv_heads + h;
  uint8_t* codes = (is_v ? p.v_codes : p.k_codes) + ((int64_t)unit.x * p.kv_heads + h) * (BS * D);
  const float s_old = live && off > 0 ? *scale : 0.f;
  float amax = 0.f, s = 1.f, inv = 1.f, shrink = 1.f;
  bool poisoned = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int i = 0; i < S::kItems; ++i) {
      const int row = row0 + i * kRowStep;
      uint8_t* dst = codes + row * D;
      if (live && row >= off && row < off + rows) {
        float x[16];
        fetch(row, x);
        if (pass == 0) {
#pragma unroll
          for (int j = 0; j < 16; ++j)   // a NaN counts as an infinity
            amax = fmaxf(amax, fabsf(x[j]) <= 3.402823466e38f ? fabsf(x[j]) : INFINITY);
        } else {
          uint2 a = make_uint2(0, 0), b = a;
          if (!poisoned) {
            a = encode8<FMT>(x, s, inv);
            b = encode8<FMT>(x + 8, s, inv);
          }
          *reinterpret_cast<uint2*>(dst + w.lo) = a;
          *reinterpret_cast<uint2*>(dst + w.hi) = b;
        }
      } else if (pass == 1 && row < off && s > s_old && !poisoned) {
        uint4 v = *reinterpret_cast<const uint4*>(dst + item * 16);
        uint32_t* c = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t y = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            y |= encode<FMT>(__fmul_rn(decode<FMT>((c[j] >> (8 * k)) & 0xffu), shrink)) << (8 * k);
          c[j] = y;
        }
        *reinterpret_cast<uint4*>(dst + item * 16) = v;
      }
    }
    if (pass == 1) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    if (S::kWarps > 1) {
      if (lane == 0) warp_max[warp] = amax;
      __syncthreads();   // and every warp has read the old scale
#pragma unroll
      for (int i = 0; i < S::kWarps; ++i) amax = fmaxf(amax, warp_max[sub * S::kWarps + i]);
    }
    if (!live) return;
    s = fmaxf(__fdiv_rn(amax, kQMax<FMT>), s_old);
    if (s == 0.f) s = 1.f;
    inv = __fdiv_rn(1.f, s);
    shrink = __fdiv_rn(s_old, s);
    poisoned = !(amax < INFINITY) || !(s_old < INFINITY);
    if (part == 0 && lane == 0) *scale = poisoned ? __int_as_float(0x7fc00000) : s;
  }
}

template <typename T, int D, int BS, int FMT>
static cudaError_t launch_append8(const AppendParams8& p, cudaStream_t stream) {
  using S = AppendShape<D, BS>;
  const int64_t ctas = (int64_t)p.units_cap * ((2 * p.kv_heads + S::kTiles - 1) / S::kTiles) +
                       (p.heads > 0 ? p.tokens : 0);
  if (ctas == 0) return cudaSuccess;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_dependent(append_kernel8<T, D, BS, FMT>, dim3((unsigned)ctas), 128, 0, stream, p);
}

template <typename T, int FMT>
static cudaError_t pick_append(const AppendParams8& p, int d, int bs, cudaStream_t stream) {
  if (d == 128) {
    if (bs == 16) return launch_append8<T, 128, 16, FMT>(p, stream);
    if (bs == 32) return launch_append8<T, 128, 32, FMT>(p, stream);
    return launch_append8<T, 128, 64, FMT>(p, stream);
  }
  if (bs == 16) return launch_append8<T, 64, 16, FMT>(p, stream);
  if (bs == 32) return launch_append8<T, 64, 32, FMT>(p, stream);
  return launch_append8<T, 64, 64, FMT>(p, stream);
}

cudaError_t launch_kv8_append(const AppendParams8& p, int d, int bs, int format, int dtype,
                              cudaStream_t stream) {
  if (dtype == kDtF16)
    return format == TKV_KV8_INT8 ? pick_append<__half, TKV_KV8_INT8>(p, d, bs, stream)
                                  : pick_append<__half, TKV_KV8_E4M3>(p, d, bs, stream);
  return format == TKV_KV8_INT8 ? pick_append<__nv_bfloat16, TKV_KV8_INT8>(p, d, bs, stream)
                                : pick_append<__nv_bfloat16, TKV_KV8_E4M3>(p, d, bs, stream);
}

}  // namespace tkv
