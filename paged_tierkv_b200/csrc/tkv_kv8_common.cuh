// tkv_kv8_common.cuh -- device helpers shared by the attention kernels over
// the 8-bit paged cache.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tkv_kv8.h"
#include "tkv_ptx.cuh"

namespace tkv {

// One request as the attention kernels see it.
struct RequestLens {
  int q0, q_len, kv;
  // Requests of up to few_rows_max query rows per kv head run in
  // few_rows_kernel, the others in many_rows_kernel.
  __device__ __forceinline__ bool few_rows(const AttnParams8& p) const {
    return q_len > 0 && (int64_t)q_len * p.group <= p.few_rows_max;
  }
  // First key that any query token sees.
  __device__ __forceinline__ int first_key(const AttnParams8& p) const {
    return p.window > 0 ? min(max(0, kv - q_len - p.window + 1), kv) : 0;
  }
};

__device__ __forceinline__ RequestLens request_lens(const AttnParams8& p, int bs, int req) {
  RequestLens n;
  n.q0 = min(max(p.cu_q[req], 0), p.tokens);
  n.q_len = min(max(p.cu_q[req + 1], n.q0), p.tokens) - n.q0;
  n.kv = min(max(p.kv_lens[req], 0), p.table_width * bs);
  return n;
}

// Two fp16 / bf16 values in a word.
__device__ __forceinline__ uint32_t pack_out(bool bf16, float a, float b) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  return pack_half2(a, b);
}
__device__ __forceinline__ float2 unpack_in(bool bf16, uint32_t w) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
  return x;
}

// a / b for a >= 0, b > 0: the 64-bit division is a subroutine of some 500
// clocks, and small steps have several in a row.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}

// Power of two that brings a row whose largest magnitude is amax into fp16
// with its maximum in [2^14, 2^15), and its inverse.
__device__ __forceinline__ void fp16_scale(float amax, float& up, float& down) {
  up = down = 1.f;
  if (!(amax > 0.f) || !(amax < INFINITY)) return;
  const int e = max((int)(__float_as_uint(amax) >> 23), 20);   // biased exponent
  up = __uint_as_float((uint32_t)(268 - e) << 23);             // 2^(14 - (e - 127))
  down = __uint_as_float((uint32_t)(e - 14) << 23);            // 2^((e - 127) - 14)
}

// 2^14 over the power of two at or above s: s times it lies in (2^13, 2^14]; for
// an s below 2^-114 2^127, the largest power of two.
__device__ __forceinline__ float scale_inverse(float s) {
  const int e = max((int)(__float_as_uint(s) >> 23), 13);
  return __uint_as_float((uint32_t)(267 - e) << 23);
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Smallest e with x <= 2^e, for a finite x > 0 (subnormal ones too).
__device__ __forceinline__ int ceil_log2(float x) {
  const uint32_t b = __float_as_uint(x);
  if (b < 0x00800000u) return (b > 1 ? 32 - __clz(b - 1) : 0) - 149;
  return (int)(b >> 23) - 127 + ((b & 0x007fffffu) != 0);
}

__device__ __forceinline__ float row_lse(float m, float sum) { return (m + lg2(sum)) * kLn2; }

// ---- codes to fp16, exact for int8 and for finite e4m3
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t cvt_e4m3x2_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}

// The word's codes 0, 1 -> lo and 2, 3 -> hi.  int8: code + 128 in the low
// byte of an fp16 with exponent 2^10 is 1152 + code.
template <int FMT>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == TKV_KV8_INT8) {
    const uint32_t x = w ^ 0x80808080u;
    lo = hsub2_u32(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
    hi = hsub2_u32(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
  } else {
    lo = cvt_e4m3x2(w);
    hi = cvt_e4m3x2_hi(w);
  }
}

// out[e] = (code e of wa, code e of wb).
template <int FMT>
__device__ __forceinline__ void expand_pairs(uint32_t wa, uint32_t wb, uint32_t (&out)[4]) {
  if (FMT == TKV_KV8_INT8) {
    out[0] = hsub2_u32((__byte_perm(wa, wb, 0x4400) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    out[1] = hsub2_u32((__byte_perm(wa, wb, 0x5511) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    out[2] = hsub2_u32((__byte_perm(wa, wb, 0x6622) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    out[3] = hsub2_u32((__byte_perm(wa, wb, 0x7733) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
  } else {
    const uint32_t x = __byte_perm(wa, wb, 0x5140), y = __byte_perm(wa, wb, 0x7362);
    out[0] = cvt_e4m3x2(x);
    out[1] = cvt_e4m3x2_hi(x);
    out[2] = cvt_e4m3x2(y);
    out[3] = cvt_e4m3x2_hi(y);
  }
}

// mbar_wait with a suspend hint: a waiting thread sleeps on the barrier instead
// of polling it, which leaves the issue slots to the others; false on timeout.
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(20000u)   // nanoseconds
        : "memory");
    if (ok) return true;
    const uint64_t now = globaltimer();
    if (t0 == 0) t0 = now;
    else if (now - t0 > kWaitTimeoutNs) return false;
  }
}

// ---- asynchronous 4-byte copies that arrive on an mbarrier
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// 16 bytes past L1; cp_async_wait_all waits for this thread's copies.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// One arrival (counted in the barrier's initial count) once this thread's
// earlier cp.async copies have landed.
__device__ __forceinline__ void cp_async_mbar_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Orders this thread's shared-memory stores before later asynchronous-proxy
// accesses (TMA writes, tcgen05.mma reads) that a barrier puts after them.
__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

}  // namespace tkv
