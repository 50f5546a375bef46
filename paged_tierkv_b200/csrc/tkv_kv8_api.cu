// tkv_kv8_api.cu -- the tkv_kv8_* and tkv_rotary_* entry points: argument
// checks, workspace layout and launches.  Nothing here allocates or throws.
#include <atomic>
#include <cmath>
#include <cstring>

#include "tkv_kv8.h"

using namespace tkv;

namespace {

inline int32_t cuda_status(cudaError_t e) { return e == cudaSuccess ? TKV_OK : TKV_ERR_CUDA; }

bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64; }

int32_t check_cache(const tkv_kv8_cache* c) {
  if (!c) return TKV_ERR_INVALID;
  if (c->format != TKV_KV8_INT8 && c->format != TKV_KV8_E4M3) return TKV_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return TKV_ERR_UNSUPPORTED;
  if (!block_size_ok(c->block_size)) return TKV_ERR_UNSUPPORTED;
  if (c->kv_heads <= 0 || c->blocks <= 0) return TKV_ERR_INVALID;
  if (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale) return TKV_ERR_INVALID;
  if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scale, 4) ||
      !aligned(c->v_scale, 4))
    return TKV_ERR_INVALID;
  if (c->blocks >= (int64_t(1) << 31) / c->block_size / c->kv_heads) return TKV_ERR_INVALID;
  return TKV_OK;
}

int32_t check_view(const tkv_token_view& v) {
  if (!v.data || !aligned(v.data, 16) || v.token_stride % 8 || v.head_stride % 8) return TKV_ERR_INVALID;
  return TKV_OK;
}

int32_t check_rotary(const tkv_rotary* r, int head_dim, bool any_token) {
  if (!r || !r->cos_sin || !aligned(r->cos_sin, 16) || r->rows <= 0) return TKV_ERR_INVALID;
  if (r->rot_dim <= 0 || r->rot_dim % 16 || r->rot_dim > head_dim) return TKV_ERR_UNSUPPORTED;
  if (r->axes < 1 || r->axes > 4) return TKV_ERR_UNSUPPORTED;
  if (r->positions_bytes != 4 && r->positions_bytes != 8) return TKV_ERR_UNSUPPORTED;
  if (any_token && (!r->positions || !aligned(r->positions, r->positions_bytes))) return TKV_ERR_INVALID;
  int64_t sum = 0;
  for (int a = 0; a < r->axes; ++a) {
    if (r->sections[a] < 0) return TKV_ERR_INVALID;
    sum += r->sections[a];
  }
  return sum == r->rot_dim / 2 ? TKV_OK : TKV_ERR_INVALID;
}

// SM count of the current device, looked up once per device.
int32_t device_sms(int* sms) {
  static std::atomic<int> known[kKv8MaxDevices];
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TKV_ERR_NO_DEVICE;
  const bool cached = dev >= 0 && dev < kKv8MaxDevices;
  if (cached && (*sms = known[dev].load(std::memory_order_relaxed)) > 0) return TKV_OK;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10 ||
      cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return TKV_ERR_NO_DEVICE;
  if (cached) known[dev].store(*sms, std::memory_order_relaxed);
  return TKV_OK;
}

int32_t check_attention(const tkv_kv8_cache* c, const tkv_kv8_attention_args* a) {
  const int32_t st = check_cache(c);
  if (st != TKV_OK) return st;
  if (!a) return TKV_ERR_INVALID;
  if (a->requests < 1 || a->requests > TKV_KV8_MAX_REQUESTS) return TKV_ERR_INVALID;
  if (a->tokens < 0 || a->heads <= 0 || a->heads % c->kv_heads) return TKV_ERR_INVALID;
  if (a->heads / c->kv_heads > 64) return TKV_ERR_UNSUPPORTED;
  if ((int64_t)a->tokens * (a->heads / c->kv_heads) >= (int64_t(1) << 26)) return TKV_ERR_UNSUPPORTED;
  if (a->dtype != TKV_DTYPE_F16 && a->dtype != TKV_DTYPE_BF16) return TKV_ERR_UNSUPPORTED;
  if (a->max_q_len < 0 || a->window < 0) return TKV_ERR_INVALID;
  if (a->table_width < 0 || a->table_stride < a->table_width ||
      (int64_t)a->table_width * c->block_size >= (int64_t(1) << 30))
    return TKV_ERR_INVALID;
  if (!(a->scaling > 0.f) || !std::isfinite(a->scaling)) return TKV_ERR_INVALID;
  return TKV_OK;
}

}  // namespace

bool tkv::kv8_code_maps(const AttnParams8& p, int d, CUtensorMap maps[2]) {
  const int64_t rows = p.blocks * p.kv_heads * p.block_size;
  const int box = p.block_size < 32 ? p.block_size : 32;
  return encode_code_map(&maps[0], p.k_codes, rows, d, box) && encode_code_map(&maps[1], p.v_codes, rows, d, box);
}

extern "C" {

int32_t tkv_kv8_plan_step(const tkv_kv8_plan_args* a, void* stream) {
  if (!a) return TKV_ERR_INVALID;
  if (!block_size_ok(a->block_size)) return TKV_ERR_UNSUPPORTED;
  if (a->requests < 1 || a->requests > TKV_KV8_MAX_REQUESTS) return TKV_ERR_INVALID;
  if (a->tokens < 0 || a->units_cap < 0 || a->table_width < 0 || a->free_capacity < 0 ||
      a->table_stride < a->table_width ||
      (int64_t)a->table_width * a->block_size >= (int64_t(1) << 30))
    return TKV_ERR_INVALID;
  if (!a->context_lens || !a->new_lens || !a->free_count || !a->kv_lens || !a->cu_q || !a->admitted ||
      !a->num_units || !a->free_count_out)
    return TKV_ERR_INVALID;
  if (a->tokens > 0 && (!a->slot_map || !a->token_request || !a->positions)) return TKV_ERR_INVALID;
  if (a->units_cap > 0 && (!a->units || !aligned(a->units, 16))) return TKV_ERR_INVALID;
  if (a->table_width > 0 && !a->block_table) return TKV_ERR_INVALID;
  if (a->free_capacity > 0 && !a->free_blocks) return TKV_ERR_INVALID;
  return cuda_status(launch_plan_step(*a, reinterpret_cast<cudaStream_t>(stream)));
}

int32_t tkv_rotary_embed(const tkv_rotary_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->heads < 0 || a->kv_heads < 0) return TKV_ERR_INVALID;
  if (a->head_dim <= 0 || a->head_dim % 16 || a->head_dim > 256) return TKV_ERR_UNSUPPORTED;
  if (a->dtype != TKV_DTYPE_F16 && a->dtype != TKV_DTYPE_BF16) return TKV_ERR_UNSUPPORTED;
  const int32_t st = check_rotary(&a->rotary, a->head_dim, a->tokens > 0);
  if (st != TKV_OK) return st;
  RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  p.rot = a->rotary;
  if (a->tokens > 0 && a->heads > 0) {
    if (check_view(a->q) != TKV_OK || check_view(a->q_out) != TKV_OK) return TKV_ERR_INVALID;
    p.q = a->q;
    p.q_out = a->q_out;
  }
  if (a->tokens > 0 && a->kv_heads > 0) {
    if (check_view(a->k) != TKV_OK || check_view(a->k_out) != TKV_OK) return TKV_ERR_INVALID;
    p.k = a->k;
    p.k_out = a->k_out;
  }
  p.err = a->error_word;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  return cuda_status(launch_rotary(p, a->dtype, reinterpret_cast<cudaStream_t>(stream)));
}

int32_t tkv_kv8_append(const tkv_kv8_cache* cache, const tkv_kv8_append_args* a, void* stream) {
  int32_t st = check_cache(cache);
  if (st != TKV_OK) return st;
  if (!a || a->tokens < 0 || a->units_cap < 0 || a->heads < 0) return TKV_ERR_INVALID;
  if (a->dtype != TKV_DTYPE_F16 && a->dtype != TKV_DTYPE_BF16) return TKV_ERR_UNSUPPORTED;
  const bool rotate = a->rotary.rot_dim != 0;
  if (a->heads > 0 && !rotate) return TKV_ERR_INVALID;
  if (rotate && (st = check_rotary(&a->rotary, cache->head_dim, a->tokens > 0)) != TKV_OK) return st;
  if (!a->num_units || (a->units_cap > 0 && (!a->units || !aligned(a->units, 16)))) return TKV_ERR_INVALID;
  if (a->tokens == 0) return TKV_OK;
  if (check_view(a->k) != TKV_OK || check_view(a->v) != TKV_OK) return TKV_ERR_INVALID;
  if (a->heads > 0 && (check_view(a->q) != TKV_OK || check_view(a->q_out) != TKV_OK)) return TKV_ERR_INVALID;
  AppendParams8 p;
  std::memset(&p, 0, sizeof(p));
  p.rot = a->rotary;
  p.has_rot = rotate;
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.q_out = a->q_out;
  p.k_codes = reinterpret_cast<uint8_t*>(cache->k_codes);
  p.v_codes = reinterpret_cast<uint8_t*>(cache->v_codes);
  p.k_scale = cache->k_scale;
  p.v_scale = cache->v_scale;
  p.units = a->units;
  p.num_units = a->num_units;
  p.err = a->error_word;
  p.blocks = cache->blocks;
  p.units_cap = a->units_cap;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = cache->kv_heads;
  return cuda_status(launch_kv8_append(p, cache->head_dim, cache->block_size, cache->format, a->dtype,
                                       reinterpret_cast<cudaStream_t>(stream)));
}

int32_t tkv_kv8_attention_workspace(const tkv_kv8_cache* cache, const tkv_kv8_attention_args* a,
                                    size_t* workspace_bytes_out) {
  int32_t st = check_attention(cache, a);
  if (st != TKV_OK) return st;
  if (!workspace_bytes_out) return TKV_ERR_INVALID;
  int sms = 0;
  if ((st = device_sms(&sms)) != TKV_OK) return st;
  size_t counters = 0, data = 0;
  kv8_attention_scratch(sms, cache->head_dim, a->heads / cache->kv_heads, a->max_q_len,
                        &counters, &data);
  *workspace_bytes_out = required_workspace(counters, data);
  return TKV_OK;
}

int32_t tkv_kv8_attention(const tkv_kv8_cache* cache, const tkv_kv8_attention_args* a, void* stream) {
  int32_t st = check_attention(cache, a);
  if (st != TKV_OK) return st;
  if (!a->kv_lens || !a->cu_q || (a->table_width > 0 && !a->block_table)) return TKV_ERR_INVALID;
  if (a->tokens == 0) return TKV_OK;
  if (check_view(a->q) != TKV_OK || !a->out || !aligned(a->out, 16)) return TKV_ERR_INVALID;
  int sms = 0;
  if ((st = device_sms(&sms)) != TKV_OK) return st;
  size_t counters = 0, data = 0;
  const int group = a->heads / cache->kv_heads;
  kv8_attention_scratch(sms, cache->head_dim, group, a->max_q_len, &counters, &data);
  if (!a->workspace || !aligned(a->workspace, 256) || !layout_fits(a->workspace_bytes, counters, data))
    return TKV_ERR_WORKSPACE;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a->workspace);
  AttnParams8 p;
  std::memset(&p, 0, sizeof(p));
  p.q = a->q;
  p.out = a->out;
  p.out_lse = a->out_lse;
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.kv_lens = a->kv_lens;
  p.cu_q = a->cu_q;
  p.k_codes = reinterpret_cast<const uint8_t*>(cache->k_codes);
  p.v_codes = reinterpret_cast<const uint8_t*>(cache->v_codes);
  p.k_scale = cache->k_scale;
  p.v_scale = cache->v_scale;
  p.err = reinterpret_cast<uint32_t*>(ws);
  p.counters = reinterpret_cast<uint32_t*>(ws + kAlign);
  p.data = ws + data_base(a->workspace_bytes);
  p.blocks = cache->blocks;
  p.requests = a->requests;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = cache->kv_heads;
  p.group = group;
  p.table_width = a->table_width;
  p.max_q_len = a->max_q_len;
  // no context reaches 2^30 keys, so a window of that many hides none; the
  // kernels' position arithmetic (keys - query tokens - window) stays in 32 bits
  p.window = a->window < (1 << 30) ? a->window : 0;
  p.scale_log2 = a->scaling * kLog2e;
  p.group_inv = group > 1 ? (uint32_t)(((uint64_t(1) << 32) + group - 1) / group) : 0;
  p.block_size = cache->block_size;
  p.bf16 = a->dtype == TKV_DTYPE_BF16;
  return cuda_status(launch_kv8_attention(p, sms, cache->head_dim, cache->format,
                                          reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
