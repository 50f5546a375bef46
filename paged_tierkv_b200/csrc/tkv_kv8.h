// tkv_kv8.h -- parameter blocks and launchers of the 8-bit paged cache's
// kernels (not part of the public ABI).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "tierkv_b200.h"
#include "tkv_internal.h"

namespace tkv {

using RotaryArgs = tkv_rotary;

constexpr int kKv8MaxDevices = 64;

// Opt-ins (more than 48 KB of shared memory, clusters of 16) are per function and
// device; `done` (one per function and opt-in) holds the devices that have it.
template <typename Kernel>
cudaError_t allow(Kernel kern, cudaFuncAttribute what, int value, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev >= 0 && dev < kKv8MaxDevices ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, what, value);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
template <typename Kernel>
cudaError_t allow_smem(Kernel kern, int bytes, std::atomic<uint64_t>& done) {
  return allow(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes, done);
}

struct RotaryParams {
  RotaryArgs rot;
  tkv_token_view q, k, q_out, k_out;
  uint32_t* err;
  int32_t tokens, heads, kv_heads, head_dim;
};

struct AppendParams8 {
  RotaryArgs rot;
  tkv_token_view k, v, q, q_out;
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* k_scale;
  float* v_scale;
  const int32_t* units;
  const int32_t* num_units;
  uint32_t* err;
  int64_t blocks;
  int32_t units_cap, tokens, heads, kv_heads;
  int32_t has_rot;
};

// A launch with programmatic dependent launch: the kernel's CTAs may start while
// the previous kernel of the stream drains, and wait for it (griddepcontrol.wait)
// before they touch memory.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                             const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, Params(args)...);
}

// A unit of many_rows_kernel split over `parts` CTAs; parts 0: none.
struct MergeUnit {
  int32_t parts, slot0;   // the first part's slot in its CTA
  int32_t q0, row0, head, rows;
};

struct AttnParams8 {
  tkv_token_view q;
  void* out;
  float* out_lse;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const float* k_scale;
  const float* v_scale;
  uint32_t* err;
  uint32_t* counters;
  uint8_t* data;
  float4* part_o;         // many_rows_kernel: [ctas][2][head_dim / 4][256]
  float* part_lse;        // [ctas][2][256], log2
  MergeUnit* merges;      // [ctas]
  int64_t blocks;
  int32_t requests, tokens, heads, kv_heads, group;
  int32_t table_width, max_q_len, window, block_size;
  int32_t bf16;          // q and out are bf16 (else fp16)
  int32_t few_rows_max;  // rows per kv head of the requests that few_rows_kernel takes
  float scale_log2;
  uint32_t group_inv;    // ceil(2^32 / group) for 1 < group <= 64
#ifdef __CUDACC__
  // row / group for a row of a request: exact for row < 2^26
  __device__ __forceinline__ int token_of(int row) const {
    return group == 1 ? row : (int)__umulhi((uint32_t)row, group_inv);
  }
#endif
};

cudaError_t launch_plan_step(const tkv_kv8_plan_args& p, cudaStream_t stream);
cudaError_t launch_rotary(const RotaryParams& p, int dtype, cudaStream_t stream);
cudaError_t launch_kv8_append(const AppendParams8& p, int head_dim, int block_size, int format,
                              int dtype, cudaStream_t stream);

// Scratch of an attention call: counters (returned to zero by the launch) and
// partial results.
void kv8_attention_scratch(int sms, int head_dim, int group, int max_q_len, size_t* counters,
                           size_t* data);
cudaError_t launch_kv8_attention(const AttnParams8& p, int sms, int head_dim, int format,
                                 cudaStream_t stream);
cudaError_t launch_many_rows(const AttnParams8& p, const CUtensorMap* maps, int sms, int head_dim, int format,
                             cudaStream_t stream);
size_t many_rows_scratch(int sms, int head_dim);
// Tensor maps of the K and V codes as [blocks * kv_heads * block_size][head_dim]
// bytes, boxes of min(block_size, 32) rows, swizzled by the row's width.
bool kv8_code_maps(const AttnParams8& p, int head_dim, CUtensorMap maps[2]);

}  // namespace tkv
