// tkv_kv8_attn.cu -- attention of a packed batch over the 8-bit paged cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tkv_kv8.h"
#include "tkv_kv8_common.cuh"

namespace tkv {

template <int FMT>
__device__ __forceinline__ float code_value(uint8_t b) {
  if (FMT == TKV_KV8_INT8) return (float)(int8_t)b;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

// One warp per (token, query head), one key at a time, online softmax.
template <int D, int FMT>
__global__ void __launch_bounds__(128) attention_simple_kernel(const AttnParams8 p) {
  const int lane = threadIdx.x & 31, bs = p.block_size;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)p.tokens * p.heads) return;
  const int t = (int)(w / p.heads), h = (int)(w % p.heads), kh = h / p.group;
  if (t < p.cu_q[0] || t >= p.cu_q[p.requests]) return;
  int lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  const RequestLens n = request_lens(p, bs, lo);
  const int pos = n.kv - (n.q0 + n.q_len - t);
  constexpr int E = D / 64;
  float2 q[E], o[E] = {};
  const uint32_t* qp = reinterpret_cast<const uint32_t*>((const uint16_t*)p.q.data + t * p.q.token_stride +
                                                         h * p.q.head_stride) + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) q[i] = unpack_in(p.bf16, qp[i]);
  float m = -INFINITY, l = 0.f;
  const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  for (int j = first; j <= pos; ++j) {
    int64_t b = p.table[lo * p.table_stride + j / bs];
    float ks = 0.f, vs = 0.f;
    if (b < 0 || b >= p.blocks) {
      b = 0;
      if (lane == 0) atomicOr(p.err, TKV_DEVERR_BAD_SLOT);
    } else {
      ks = p.k_scale[b * p.kv_heads + kh];
      vs = p.v_scale[b * p.kv_heads + kh];
    }
    const int64_t at = ((b * p.kv_heads + kh) * bs + j % bs) * D + lane * 2 * E;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i)
      s += q[i].x * code_value<FMT>(p.k_codes[at + 2 * i]) + q[i].y * code_value<FMT>(p.k_codes[at + 2 * i + 1]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    s *= ks * p.scale_log2;
    const float mn = fmaxf(m, s);
    const float a = exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * a + e;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      o[i].x = o[i].x * a + e * vs * code_value<FMT>(p.v_codes[at + 2 * i]);
      o[i].y = o[i].y * a + e * vs * code_value<FMT>(p.v_codes[at + 2 * i + 1]);
    }
  }
  uint32_t* op = reinterpret_cast<uint32_t*>((uint16_t*)p.out + w * D) + lane * E;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) op[i] = pack_out(p.bf16, o[i].x * inv, o[i].y * inv);
  if (p.out_lse && lane == 0) p.out_lse[w] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

void kv8_attention_scratch(int, int, int, int, int, int, size_t* counters, size_t* data) {
  *counters = 0;
  *data = 0;
}

cudaError_t launch_kv8_attention(const AttnParams8& p, int, int d, int format, cudaStream_t stream) {
  const unsigned grid = (unsigned)(((int64_t)p.tokens * p.heads + 3) / 4);
  if (d == 128) {
    if (format == TKV_KV8_INT8) attention_simple_kernel<128, TKV_KV8_INT8><<<grid, 128, 0, stream>>>(p);
    else attention_simple_kernel<128, TKV_KV8_E4M3><<<grid, 128, 0, stream>>>(p);
  } else {
    if (format == TKV_KV8_INT8) attention_simple_kernel<64, TKV_KV8_INT8><<<grid, 128, 0, stream>>>(p);
    else attention_simple_kernel<64, TKV_KV8_E4M3><<<grid, 128, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace tkv
