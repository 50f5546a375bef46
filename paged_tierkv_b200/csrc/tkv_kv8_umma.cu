// tkv_kv8_umma.cu -- attention over the 8-bit paged cache for requests with
// many query rows (prompts, prompt chunks), on the tcgen05 tensor cores.
//
// Rows (query token, query head of a kv head's group) are packed into units of
// 256, two 128-row query tiles that share every K/V tile of 128 tokens.  Per
// tile the CTA does S_i = Q_i K^T and O_i += P_i V (i = 0, 1), fp16 in, fp32
// out, all four accumulators in tensor memory:
//   columns [0, 128) S0, [128, 256) S1, [256, 256 + D) O0, [256 + D, 256 + 2 D) O1,
// the fp16 P_i of 64 tokens overwriting the first half of their S_i and feeding
// the MMA from there.
// While the tensor core works for one query tile the other one's softmax runs.
// A prompt of 8192 tokens, 32 / 8 heads of 128: 675 us, 814 TFLOP/s (from a
// graph, in runs of some 10 ms; 696-708 us under the power limit).  Bound by
// shared memory, which the MMAs of S alone read at its full bandwidth and the
// expansion writes, and by the tensor-memory reads of the softmax.
//
//   warps 0-7, 8-15  softmax of query tile 0, 1: two threads per row, 64 columns
//                    each, that exchange their maxima; also load Q and write the
//                    output (one thread a row left the softmax of a tile at twice
//                    the time of its MMAs: 691 us against 686 for the
//                    8192-token prompt, 678 against 668 with e4m3 codes)
//   warps 16-19      expand codes to fp16 (exact) and store them in the
//                    128-byte-swizzled layout that the MMA descriptors name:
//                    K as K-major rows, V as rows of the MN-major B operand
//   warp 20          issues the MMAs
//   warp 21          walks the block table: TMA boxes of codes and the scales,
//                    a tile ahead of the expansion
//
// Three kinds of code share the SM's instruction caches, and each tile passes
// through all of it: the loops over a tile's columns and over the MMAs of a
// product stay rolled (unrolled, the instruction fetch of every role stalled:
// 1141 us against 807 for the 8192-token prompt at that stage).
//
// Scales.  A tile's K scales multiply the logits of their 16 columns in fp32.
// V's go into the exponent: P' = exp2(s - m + 12 + log2(vs / 2^E)), 2^E the power
// of two at or above the largest V scale of the segment so far.  O is in units
// of 2^(E - 12) and is rescaled when E grows; the row sum gets p back by one
// multiplication with 2^E / vs per 16 columns and is in units of 2^-12 whatever
// E is, so it neither passes fp32's range nor loses a key for the sake of V's
// scales.  m follows the running maximum lazily: O is only rescaled when it has
// grown by more than 3.9 (log2; by more than 2 the 8192-token prompt takes 8 %
// longer).  With vs / 2^E at most 1, P' stays below fp16's largest number and
// normal down to 2^-25 of the row's largest.  A scale below 2^-60 of 2^E (or 0)
// is beyond what P' can hold: its keys count in the row sum, its values as
// zeros.  bf16 queries become fp16 by a power of two per row.
//
// Work is a flat list of (unit, K/V tile), where a unit counts kUnitCost tiles
// more than it has (loading Q, writing the output), cut evenly over the CTAs,
// so that causal and ragged batches and few rows over a long cache load every
// SM alike.  A unit that ends up on several CTAs leaves its partial rows (max,
// sum, accumulator) in the workspace, and merge_rows_kernel joins them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "tkv_kv8_common.cuh"

namespace tkv {

constexpr int kManyThreads = 704;
constexpr int kUnitRows = 256;
constexpr int kTok = 128;                 // tokens of a K/V tile
constexpr int kGroups = kTok / 16;        // scale groups of a tile
constexpr int kScStride = kGroups + 1;    // and (E, first token, first and last key)
constexpr int kUnitCost = 4;              // a unit's fixed cost in tiles
constexpr uint32_t kManyTmem = 512;
constexpr float kVLog = 12.f;             // log2 of P' at the row's reference and the scale 2^E
constexpr float kVLeast = 0x1p-60f;       // smallest vs / 2^E whose values count
constexpr float kLazy = 3.9f;             // growth of the maximum (log2) that P' absorbs

template <int D>
struct ManyLayout {
  static constexpr int kTile = kTok * D * 2;              // fp16 tile: [D / 64][128][64]
  static constexpr int kQOff = 0;                         // [2]
  static constexpr int kKOff = 2 * kTile;                 // [2] stages
  static constexpr int kVOff = 4 * kTile;                 // [2] stages
  static constexpr int kCodes = kTok * D;                 // staged codes of a tile
  static constexpr int kStOff = 6 * kTile;                // K, V
  static constexpr int kScOff = kStOff + 2 * kCodes;      // [4][kScStride] float4 (ks, vs, log2 (vs / 2^E), 2^E / vs)
  static constexpr int kBarOff = kScOff + 4 * kScStride * 16;
  static constexpr int kNumBars = 26;
  static constexpr int kRowOff = kBarOff + kNumBars * 8;  // [2 tiles][2 halves][128] floats: the rows'
                                                          // logit scales, then what their threads exchange
  static constexpr int kMiscOff = kRowOff + 2 * kUnitRows * 4;
  static constexpr int kBytes = kMiscOff + 128;
};
static_assert(ManyLayout<128>::kBytes <= 232448, "shared memory");

// ---- the flat list of (request, row tile, kv head) units and their K/V tiles
struct ManyUnit {
  int req, rt, head;
  int q0, q_len, kv;
  int rts;          // row tiles of the request
  int req_lo;       // first key that any of its tokens sees
  int tile0, n;     // first K/V tile, tiles of the unit
};

__device__ __forceinline__ void unit_tiles(const AttnParams8& p, ManyUnit& u) {
  const int first = p.token_of(u.rt * kUnitRows);
  const int last = min(u.q_len - 1, p.token_of(u.rt * kUnitRows + kUnitRows - 1));
  const int hi = max(0, u.kv - u.q_len + last + 1);
  const int lo = p.window > 0 ? min(max(0, u.kv - u.q_len + first + 1 - p.window), hi) : 0;
  u.tile0 = lo / kTok;
  u.n = max(1, (hi + kTok - 1) / kTok - u.tile0);   // one empty tile writes the zeros of unseen rows
}

__device__ __forceinline__ bool load_many(const AttnParams8& p, int req, ManyUnit& u) {
  const RequestLens n = request_lens(p, p.block_size, req);
  u.req = req;
  u.q0 = n.q0;
  u.q_len = n.q_len;
  u.kv = n.kv;
  u.req_lo = n.first_key(p);
  u.rts = n.q_len == 0 || n.few_rows(p) ? 0 : (int)(((int64_t)n.q_len * p.group + kUnitRows - 1) / kUnitRows);
  return u.rts > 0;
}

// A request's places in the flat list, evaluated by `lanes` threads (a power of
// two, neighbours) together; every one of them gets the sum.
__device__ __forceinline__ int64_t many_places(const AttnParams8& p, int req, int sub, int lanes) {
  ManyUnit u;
  int64_t sum = 0;
  if (req < p.requests && load_many(p, req, u))
    for (u.rt = sub; u.rt < u.rts; u.rt += lanes) {
      unit_tiles(p, u);
      sum += u.n + kUnitCost;
    }
  for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(~0u, sum, o);
  return sum * p.kv_heads;
}

__device__ __forceinline__ void next_many(const AttnParams8& p, ManyUnit& u) {
  if (++u.head < p.kv_heads) return;
  u.head = 0;
  if (++u.rt < u.rts) {
    unit_tiles(p, u);
    return;
  }
  u.rt = 0;
  for (int r = u.req + 1; r < p.requests; ++r)
    if (load_many(p, r, u)) break;
  unit_tiles(p, u);
}

// A CTA's walk over the segments of its range, each inside one unit.  A unit
// takes kUnitCost + n places of the flat list: its tiles are the last n, so a
// range that ends before them has none of the unit.
// Places are relative to the start of the CTA's range, [0, end).
struct Walk {
  ManyUnit u;
  int u_at, end;
  __device__ __forceinline__ int tiles_at() const { return u_at + kUnitCost; }
  __device__ __forceinline__ int u_end() const { return tiles_at() + u.n; }
  __device__ __forceinline__ bool more() const { return tiles_at() < end; }
  __device__ __forceinline__ int skipped() const { return max(0, -tiles_at()); }
  __device__ __forceinline__ int first() const { return u.tile0 + skipped(); }
  __device__ __forceinline__ int count() const { return min(end, u_end()) - tiles_at() - skipped(); }
  __device__ __forceinline__ bool whole() const { return tiles_at() >= 0 && end >= u_end(); }
  __device__ __forceinline__ int slot() const { return u_at <= 0 ? 0 : 1; }
  __device__ __forceinline__ int rows(const AttnParams8& p) const {
    return min(kUnitRows, u.q_len * p.group - u.rt * kUnitRows);
  }
  __device__ __forceinline__ void next(const AttnParams8& p) {
    u_at = u_end();
    if (u_at < end) next_many(p, u);
  }
};

// ---- tcgen05 helpers
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_wait_into(uint32_t (&v)[32]) {
  // the wait "rewrites" the registers, so no use of them moves above it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                 "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]),
                 "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]),
                 "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]),
                 "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&v)[32]) {
  tmem_ld32(taddr, v);
  tmem_wait_into(v);
}

// D[tmem] (+)= A[smem] * B[smem]^T, the descriptors as their two words.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                        uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem, fp16 pairs along the columns] * B[smem].
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of the MN-major B operand V: rows of 128 bytes (64 fp16 of N) with
// 128-byte swizzle, groups of 8 rows (K) 1024 bytes apart (stride offset), the
// next 64 of N a whole [128][64] panel further (leading offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(kTok * 128 >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// 32 logits of a row: those at or past `over` or below `under` become -inf, the
// others take their 16-column group's factor.
__device__ __forceinline__ void hide(uint32_t (&v)[32], int over, int under, float f0, float f1) {
#pragma unroll
  for (int x = 0; x < 32; ++x)
    v[x] = x < over && x >= under ? __float_as_uint(__uint_as_float(v[x]) * (x < 16 ? f0 : f1)) : 0xff800000u;
}

template <int D, int FMT>
__global__ void __launch_bounds__(kManyThreads, 1)
    many_rows_kernel(const __grid_constant__ AttnParams8 p, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v) {
  using L = ManyLayout<D>;
  extern __shared__ __align__(1024) uint8_t many_smem[];
  uint8_t* smem = many_smem;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* q_full = bars;          // [2] 8 warps: Q_i stored
  uint64_t* s_full = bars + 2;      // [2] S_i written (commit)
  uint64_t* p_full = bars + 4;      // [2] 8 warps: P_i stored, S_i read, O_i rescaled
  uint64_t* o_full = bars + 6;      // [2] O_i updated (commit)
  uint64_t* k_full = bars + 8;      // [2] 4 warps
  uint64_t* k_empty = bars + 10;    // [2] commit
  uint64_t* v_full = bars + 12;     // [2] 4 warps
  uint64_t* v_empty = bars + 14;    // [2] commit
  uint64_t* sc_full = bars + 16;    // [4] a tile's scales (reused 4 tiles later)
  uint64_t* done = bars + 20;
  uint64_t* st_full = bars + 21;    // [2] K, V codes staged (TMA)
  uint64_t* st_empty = bars + 23;   // [2] 4 warps
  float* row_s = reinterpret_cast<float*>(smem + L::kRowOff);
  float4* scales = reinterpret_cast<float4*>(smem + L::kScOff);
  int64_t* misc = reinterpret_cast<int64_t*>(smem + L::kMiscOff);
  MergeUnit* merge_s = reinterpret_cast<MergeUnit*>(smem + L::kMiscOff + 104);
  uint32_t* taddr_s = reinterpret_cast<uint32_t*>(smem + L::kMiscOff + 96);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 8);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 8);
      mbar_init(o_full + i, 1);
      mbar_init(k_full + i, 4);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 4);
      mbar_init(v_empty + i, 1);
      mbar_init(st_full + i, 1);
      mbar_init(st_empty + i, 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(sc_full + i, 1);
    mbar_init(done, 1);
    fence_mbar_init();
    *merge_s = MergeUnit{};
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }

  pdl_launch_dependents();
  pdl_wait();   // everything below reads what the kernels before may have written

  // ---- this CTA's range of the flat list
  Walk walk;
  {
    // 256 threads, `lanes` of them for each request of a round
    constexpr int kScan = 256;
    const int tid = threadIdx.x;
    int lanes = 32;
    while (lanes > 1 && lanes * p.requests > kScan) lanes >>= 1;
    const int sub = tid & (lanes - 1), per_round = kScan / lanes;
    const bool scans = tid < kScan;
    // most steps have a thread for every row tile: one scan finds the tile
    ManyUnit own;
    own.rts = 0;
    const int own_req = tid / lanes;
    if (scans && own_req < p.requests) load_many(p, own_req, own);
    own.rt = sub;
    if (sub < own.rts) unit_tiles(p, own);
    const int64_t mine = sub < own.rts ? (int64_t)(own.n + kUnitCost) * p.kv_heads : 0;
    const bool one_scan = !__syncthreads_or(per_round < p.requests || own.rts > lanes);
    int64_t total = 0, begin, ctas;
    auto share = [&]() {            // this CTA's part of the list; false without one
      ctas = min((int64_t)gridDim.x, total);
      if (blockIdx.x >= ctas) {
        if (tid == 0) p.merges[blockIdx.x].parts = 0;
        return false;               // CTA-uniform
      }
      begin = quotient(total * blockIdx.x, ctas);
      walk.end = (int)(quotient(total * (blockIdx.x + 1), ctas) - begin);
      return true;
    };
    if (one_scan) {
      int64_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += x;
      }
      if (scans && lane == 31) misc[warp] = inc;
      __syncthreads();
      int64_t first = inc - mine;
      for (int w = 0; w < kScan / 32; ++w) {
        if (w < warp) first += misc[w];
        total += misc[w];
      }
      if (!share()) return;
      __syncthreads();
      if (first <= begin && begin < first + mine) {
        misc[0] = first;
        misc[1] = own.req;
        misc[2] = own.rt;
        misc[3] = total;
      }
    } else {
      int64_t sum = 0;
      for (int r = tid / lanes; scans && r - tid / lanes < p.requests; r += per_round) {
        const int64_t n = many_places(p, r, sub, lanes);
        if (sub == 0) sum += n;
      }
      sum = warp_sum(sum);
      if (scans && lane == 0) misc[warp] = sum;
      __syncthreads();
      for (int w = 0; w < kScan / 32; ++w) total += misc[w];
      if (!share()) return;
      // the request that holds `begin`, then its row tile
      __syncthreads();
      int64_t at = 0;
      for (int r0 = 0; r0 < p.requests; r0 += per_round) {
        const int64_t n = scans ? many_places(p, r0 + tid / lanes, sub, lanes) : 0;
        int64_t inc = sub == 0 && scans ? n : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(~0u, inc, o);
          if (lane >= o) inc += x;
        }
        if (scans && lane == 31) misc[warp] = inc;
        __syncthreads();
        int64_t first = at + inc - n, next = at;
        for (int w = 0; w < kScan / 32; ++w) {
          if (w < warp) first += misc[w];
          next += misc[w];
        }
        if (scans && sub == 0 && first <= begin && begin < first + n) {
          misc[8] = first;
          misc[9] = r0 + tid / lanes;
        }
        __syncthreads();
        at = next;
        if (begin < at) break;      // CTA-uniform
      }
      if (warp == 0) {
        ManyUnit u;
        load_many(p, (int)misc[9], u);
        int64_t first = misc[8];
        for (int rt0 = 0;; rt0 += 32) {
          u.rt = min(rt0 + lane, u.rts - 1);
          unit_tiles(p, u);
          int64_t inc = rt0 + lane < u.rts ? (int64_t)(u.n + kUnitCost) * p.kv_heads : 0;
          const int64_t n = inc;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += x;
          }
          const int64_t here = first + inc - n;
          if (here <= begin && begin < here + n) {
            misc[0] = here;
            misc[1] = u.req;
            misc[2] = u.rt;
            misc[3] = total;
          }
          first += __shfl_sync(~0u, inc, 31);
          if (begin < first) break;
        }
      }
    }
    __syncthreads();
    load_many(p, (int)misc[1], walk.u);
    walk.u.rt = (int)misc[2];
    unit_tiles(p, walk.u);
    walk.u.head = (int)quotient(begin - misc[0], walk.u.n + kUnitCost);
    walk.u_at = (int)(misc[0] + (int64_t)walk.u.head * (walk.u.n + kUnitCost) - begin);
  }
  if (warp == 20) tmem_alloc(taddr_s, kManyTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *taddr_s;
  bool ok = true;

  if (warp == 20) {
    if (lane == 0) {
      // ---- MMA issuer
      constexpr uint32_t kIdescQK = umma_idesc_f16_f32(128, kTok);
      constexpr uint32_t kIdescPV = umma_idesc_f16_f32(128, D) | (1u << 16);   // B is MN-major
      const uint32_t base = smem_u32(smem);
      auto wait = [&](uint64_t* bar, int phase) {
        if (ok && !bounded_wait(bar, (uint32_t)(phase & 1))) ok = false;
      };
      // descriptors differ in their low words (start addresses in 16-byte units):
      // steps of 16 elements move by 2 inside a 64-element panel (K-major Q, K)
      // and by 128 (16 rows of the MN-major V)
      const uint64_t k_major = umma_desc_k_sw128(base), mn_major = umma_desc_mn_sw128(base);
      const uint32_t k_hi = (uint32_t)(k_major >> 32), mn_hi = (uint32_t)(mn_major >> 32);
      const uint32_t q_lo = (uint32_t)k_major + (L::kQOff >> 4), k_lo = (uint32_t)k_major + (L::kKOff >> 4);
      const uint32_t v_lo = (uint32_t)mn_major + (L::kVOff >> 4);
      auto qk = [&](int i, int s) {
        const uint32_t a = q_lo + i * (L::kTile >> 4), b = k_lo + s * (L::kTile >> 4), d = tmem + i * kTok;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t step = (ks >> 2) * (kTok * 128 >> 4) + (ks & 3) * 2;
          umma_ss(d, a + step, k_hi, b + step, k_hi, kIdescQK, ks > 0);
        }
        umma_commit(s_full + i);
      };
      auto pv = [&](int i, int s, bool first) {
        const uint32_t a = tmem + i * kTok, b = v_lo + s * (L::kTile >> 4), d = tmem + 256 + i * D;
#pragma unroll
        for (int ks = 0; ks < kTok / 16; ++ks)
          umma_ts(d, a + (ks >> 2) * 64 + (ks & 3) * 8, b + ks * (2048 >> 4), mn_hi, kIdescPV, ks > 0 || !first);
        umma_commit(o_full + i);
      };
      int g = 0, g1 = 0;            // tiles done before this segment; query tile 1's
      int seg = 0, seg1 = 0;
      for (Walk w = walk; w.more() && ok; w.next(p)) {
        const int n = w.count();
        const int tiles = w.rows(p) > 128 ? 2 : 1;
        // step j: O_i of tile j - 1, then S_i of tile j, for both query tiles
#pragma unroll 1
        for (int j = 0; j <= n && ok; ++j) {
          const int at = g + j;
#pragma unroll 1
          for (int i = 0; i < tiles && ok; ++i) {
            if (i == 0) {
              if (j > 0) wait(v_full + ((at - 1) & 1), (at - 1) >> 1);
              if (j < n) wait(k_full + (at & 1), at >> 1);
            }
            if (j > 0) wait(p_full + i, (i ? g1 : g) + j - 1);
            else wait(q_full + i, i ? seg1 : seg);
            tc_fence_after();
            if (!ok) break;
            if (j > 0) pv(i, (at - 1) & 1, j == 1);
            if (j < n) qk(i, at & 1);
          }
          if (!ok) break;
          if (j > 0) umma_commit(v_empty + ((at - 1) & 1));
          if (j < n) umma_commit(k_empty + (at & 1));
        }
        g += n;
        ++seg;
        if (tiles == 2) {
          g1 += n;
          ++seg1;
        }
      }
      umma_commit(done);            // every MMA issued above has completed once this phase does
      ok = bounded_wait(done, 0) && ok;
    }
    __syncwarp();
  } else if (warp == 21) {
    // ---- codes by TMA, scales through shared memory
    const int bs_log2 = 31 - __clz(p.block_size);
    const int box = min(p.block_size, 32), boxes = kTok / box;
    const int grp = lane & (kGroups - 1);                 // this lane's 16-token group
    const int box_grp = (lane & (boxes - 1)) * (box / 16);   // and its box's first group
    Walk w = walk;
    int j = 0, i = 0, cell = 0;
    float ks = 0.f, vs = 0.f, run_top = 0.f;
    bool first = false;                                   // a segment's first tile
    int tok0 = 0, lo = 0, hi = 0, head = 0;               // of the tile whose cells are held
    bool seen = false;                                    // the lane's group holds keys of the unit
    auto load = [&]() {
      if (!w.more()) return;
      tok0 = (w.first() + i) * kTok;
      first = i == 0;
      lo = w.u.req_lo;
      hi = w.u.kv;
      head = w.u.head;
      const int tok = tok0 + grp * 16;
      seen = tok + 15 >= lo && tok < hi;
      cell = seen ? p.table[w.u.req * p.table_stride + (tok >> bs_log2)] : 0;
      const bool good = cell >= 0 && cell < p.blocks;
      if (seen && !good) atomicOr(p.err, TKV_DEVERR_BAD_SLOT);
      ks = vs = 0.f;
      if (!good) cell = -1;
      else if (seen) {
        ks = p.k_scale[(int64_t)cell * p.kv_heads + head];
        vs = p.v_scale[(int64_t)cell * p.kv_heads + head];
      }
      if (++i == w.count()) {
        w.next(p);
        i = 0;
      }
    };
    bool more = w.more();
    load();
    for (; more; ++j) {
      // the segment's largest V scale so far; a NaN does not move E
      float top = vs <= 0x1p127f ? vs : 0.f;
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
      run_top = fmaxf(first ? 0.f : run_top, top);
      const int e = run_top > 0.f ? ceil_log2(run_top) : 0;
      // a group without a V scale to speak of (0: nothing stored, a bad slot)
      // has its codes zeroed, and takes a scale that is as good as any
      float v1 = vs * exp2_int((-e) >> 1) * exp2_int(-e - ((-e) >> 1));   // exact, or far below kVLeast
      const bool none = fabsf(v1) < kVLeast;
      if (none) v1 = 1.f;
      float4* sc = scales + (j & 3) * kScStride;
      if (lane < kGroups) sc[lane] = make_float4(ks, none ? 0.f : vs, lg2(v1), 1.f / v1);
      if (lane == 0)
        sc[kGroups] = make_float4((float)e, __int_as_float(tok0), __int_as_float(lo), __int_as_float(hi));
      __syncwarp();
      if (lane == 0) mbar_arrive(sc_full + (j & 3));
      const uint32_t live = __ballot_sync(~0u, seen) & ((1u << kGroups) - 1);
      const uint32_t mask = ((1u << (box / 16)) - 1);
      const bool load_box = lane < boxes && (live >> box_grp & mask);
      const uint32_t bytes = __popc(__ballot_sync(~0u, load_box)) * box * D;
      // a box's block: that of its first group with keys
      const int src = box_grp + (load_box ? __ffs(live >> box_grp & mask) - 1 : 0);
      const int blk = __shfl_sync(~0u, cell, src);
      // a bad slot's box lies before the cache, which TMA fills with zeros
      const int y = blk < 0 ? -box : ((blk * p.kv_heads + head) << bs_log2) + ((box_grp * 16) & (p.block_size - 1));
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        // one lane's timeout is the warp's: what the boxes announce is what they load
        ok = __all_sync(~0u, ok && bounded_wait(st_empty + kv, (uint32_t)(j & 1) ^ 1));
        if (lane == 0 && ok) mbar_arrive_expect_tx(st_full + kv, bytes);
        __syncwarp();
        if (load_box && ok)
          tma_load_2d(smem + L::kStOff + kv * L::kCodes + (box_grp * 16) * D, kv ? &tm_v : &tm_k, 0, y, st_full + kv);
      }
      more = w.more();
      load();
    }
    // no copy may still be landing when the CTA exits
    if (j > 0)
      for (int kv = 0; kv < 2; ++kv)
        if (!bounded_wait(st_full + kv, (uint32_t)((j - 1) & 1))) ok = false;
    __syncwarp();
  } else if (warp >= 16) {
    // ---- codes -> fp16 tiles
    constexpr int kPerRow = D / 16;              // 16-byte chunks of a row of codes
    constexpr int kPassRows = 128 / kPerRow;     // rows that 128 threads x 16 bytes cover
    const int t = threadIdx.x - 512;
    // chunk of the row and row of the pass: the eight lanes of a store phase hold
    // four chunks of two neighbouring rows of one 64-element panel, which the
    // swizzle spreads over all banks
    const int c16 = (t & 3) + (kPerRow == 8 ? ((t >> 4) & 1) * 4 : 0);
    const int row = kPerRow == 8 ? ((t >> 2) & 3) + (t >> 5) * 4 : t >> 2;
    const uint32_t from = swz<kPerRow == 8 ? 7 : 3>((uint32_t)(row * D + c16 * 16));
    const int c = 2 * (c16 & 3);
    const uint32_t to0 = ((c16 >> 2) * kTok + row) * 128 + ((c ^ (row & 7)) << 4);
    const uint32_t to1 = ((c16 >> 2) * kTok + row) * 128 + (((c + 1) ^ (row & 7)) << 4);
    int n = 0;
    for (Walk w = walk; w.more(); w.next(p)) n += w.count();
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int s = j & 1;
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        if (ok && !bounded_wait(st_full + kv, (uint32_t)(j & 1))) ok = false;
        if (ok && !bounded_wait((kv ? v_empty : k_empty) + s, (uint32_t)((j >> 1) & 1) ^ 1)) ok = false;
        const float4 info = scales[(j & 3) * kScStride + kGroups];
        const int tok = __float_as_int(info.y) + row, lo = __float_as_int(info.z), hi = __float_as_int(info.w);
        const uint8_t* src = smem + L::kStOff + kv * L::kCodes + from;
        uint8_t* dst = smem + (kv ? L::kVOff : L::kKOff) + s * L::kTile;
        // rows of a pass are kPassRows (a multiple of 8) apart: the swizzles repeat
#pragma unroll 2
        for (int i = 0; i < kPerRow; ++i) {
          uint4 x = *reinterpret_cast<const uint4*>(src + i * kPassRows * D);
          // rows that nobody sees may hold anything
          if (tok + i * kPassRows < lo || tok + i * kPassRows >= hi ||
              (kv && scales[(j & 3) * kScStride + (row + i * kPassRows) / 16].y == 0.f))
            x = make_uint4(0, 0, 0, 0);
          uint4 f[2];
          expand4<FMT>(x.x, f[0].x, f[0].y);
          expand4<FMT>(x.y, f[0].z, f[0].w);
          expand4<FMT>(x.z, f[1].x, f[1].y);
          expand4<FMT>(x.w, f[1].z, f[1].w);
          *reinterpret_cast<uint4*>(dst + to0 + i * kPassRows * 128) = f[0];
          *reinterpret_cast<uint4*>(dst + to1 + i * kPassRows * 128) = f[1];
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive((kv ? v_full : k_full) + s);
          mbar_arrive(st_empty + kv);
        }
      }
    }
  } else {
    // ---- softmax: threads t of halves 0 and 1 own row t of query tile i, and of
    // it the columns [64 half, 64 half + 64) of S and half of the columns of O
    const int i = warp >> 3, half = (warp >> 2) & 1;
    const int t = threadIdx.x & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t s_col = lane_base + i * kTok + half * 64;
    const uint32_t o_col = lane_base + 256 + i * D + half * (D / 2);
    float* row_scale = row_s + i * 256;                         // [128]
    float* mine = row_s + i * 256 + half * 128 + t;             // exchanged with the row's other thread
    const float* other = row_s + i * 256 + (half ^ 1) * 128 + t;
    uint8_t* q_tile = smem + L::kQOff + i * L::kTile;
    const bool bf16 = p.bf16 != 0;
    auto wait = [&](uint64_t* bar, int phase) {
      if (ok && !bounded_wait(bar, (uint32_t)(phase & 1))) ok = false;
    };
    int tile = 0;                   // tiles of the walk before this one (scale slots)
    int at = 0;                     // tiles this query tile has done
    for (Walk w = walk; w.more(); w.next(p)) {
      const int n = w.count(), rows = w.rows(p);
      if (i * 128 >= rows) {        // tile 1 of a unit of up to 128 rows
        tile += n;
        continue;
      }
      // Q rows of this warp -> fp16, K-major 128-byte-swizzled; kRowLanes lanes a row
      constexpr int kRowLanes = D / 8;
      const int row0 = w.u.rt * kUnitRows + i * 128;   // the tile's first row within the request
      const int wrow = (warp & 7) * 16;
      {
        const int ch = lane % kRowLanes;
        uint8_t* line = q_tile + (ch >> 3) * (kTok * 128);
#pragma unroll 1
        for (int c = 0; c < 16; c += 32 / kRowLanes) {
          const int tr = wrow + c + lane / kRowLanes;
          const int urow = min(row0 + tr, w.u.q_len * p.group - 1);
          const int tok = p.token_of(urow);
          cp_async16(line + tr * 128 + (((ch & 7) ^ (tr & 7)) << 4),
                     (const uint16_t*)p.q.data + (w.u.q0 + tok) * p.q.token_stride +
                         (int64_t)(w.u.head * p.group + urow - tok * p.group) * p.q.head_stride + ch * 8);
        }
        cp_async_wait_all();
        float down = 1.f;
        if (bf16) {
#pragma unroll 4
          for (int c = 0; c < 16; c += 32 / kRowLanes) {
            const int tr = wrow + c + lane / kRowLanes;
            uint4* at = reinterpret_cast<uint4*>(line + tr * 128 + (((ch & 7) ^ (tr & 7)) << 4));
            uint4 v = *at;             // this lane's own copy
            uint32_t* x = reinterpret_cast<uint32_t*>(&v);
            float2 f[4];
            float amax = 0.f, up;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              f[k] = unpack_in(true, x[k]);
              amax = fmaxf(amax, fmaxf(fabsf(f[k].x), fabsf(f[k].y)));
            }
#pragma unroll
            for (int o = kRowLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
            fp16_scale(amax, up, down);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = pack_half2(f[k].x * up, f[k].y * up);
            *at = v;
            if (ch == 0) row_scale[tr] = p.scale_log2 * down;
          }
        } else if (lane < 16) {
          row_scale[wrow + lane] = p.scale_log2;
        }
      }
      fence_proxy_async();
      tc_fence_before();
      named_barrier(1 + i, 256);
      const float rscale = row_scale[t];
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + i);
      const int r = i * 128 + t;
      const bool live = r < rows;
      const int urow = min(row0 + t, w.u.q_len * p.group - 1);
      const int tok = p.token_of(urow);
      const int hi = w.u.kv - w.u.q_len + tok + 1;            // keys [lo, hi) are visible
      const int lo = p.window > 0 ? hi - p.window : 0;
      // every row of the warp sees keys [all_lo, all_hi)
      const int all_hi = __shfl_sync(~0u, hi, 0), all_lo = __shfl_sync(~0u, lo, 31);
      float m = -INFINITY, l = 0.f;       // reference of the exponents (log2), sum in units of 2^-kVLog
      float e_v = 0.f;                    // E
      const int tile0 = w.first();
      for (int j = 0; j < n; ++j, ++at, ++tile) {
        const float4* sc = scales + (tile & 3) * kScStride + half * 4;
        wait(s_full + i, at);
        wait(sc_full + (tile & 3), tile >> 2);   // complete by now: orders the scales' reads
        __syncwarp();
        tc_fence_after();
        const int k0 = (tile0 + j) * kTok + half * 64;          // this thread's first key
        const bool edge = k0 + 64 > all_hi || k0 < all_lo;
        // pass 1: the row's maximum
        float mx = -INFINITY;
        uint32_t dead = 0;                  // edge tiles: groups that the row does not see
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32];
          tmem_load(s_col + c * 32, v);
          if (edge) hide(v, hi - (k0 + c * 32), lo - (k0 + c * 32), 1.f, 1.f);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a = __uint_as_float(v[h * 16]), a2 = __uint_as_float(v[h * 16 + 1]);
#pragma unroll
            for (int k = 2; k < 14; k += 4) {
              a = max3(a, __uint_as_float(v[h * 16 + k]), __uint_as_float(v[h * 16 + k + 1]));
              a2 = max3(a2, __uint_as_float(v[h * 16 + k + 2]), __uint_as_float(v[h * 16 + k + 3]));
            }
            a = fmaxf(max3(a, __uint_as_float(v[h * 16 + 14]), __uint_as_float(v[h * 16 + 15])), a2);
            // an unseen group's scale does not count (0 or NaN where nothing is stored)
            if (edge && a == -INFINITY) dead |= 1u << (c * 2 + h);
            else mx = fmaxf(mx, a * sc[c * 2 + h].x);
          }
        }
        // the row's other half; it reads this before the next tile's S is there
        *mine = mx;
        named_barrier(1 + i, 256);
        mx = fmaxf(mx, *other);
        mx *= rscale;
        // V's power of two: set by the first tile, moved when a scale outgrows it
        float shift = 0.f;                            // log2 of the factor that O takes
        const float e_tile = sc[kGroups - half * 4].x;
        if (j > 0) shift = e_v - e_tile;
        e_v = e_tile;
        if (mx > m + kLazy) {
          if (m != -INFINITY) {                       // nothing summed yet: nothing to rescale
            shift += m - mx;
            l *= ex2(m - mx);
          }
          m = mx;
        }
        if (__any_sync(~0u, shift != 0.f)) {
          const float f = ex2(shift);
          wait(o_full + i, at - 1);
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[16];
            tmem_load16(o_col + c * 16, o);
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st16(o_col + c * 16, o);
          }
        }
        const float off = kVLog - (m == -INFINITY ? 0.f : m);
        // pass 2: P' and the sum
        auto probabilities = [&](int c, uint32_t(&v)[32]) {
          uint32_t pk[16];
          const float4 g[2] = {sc[c * 2], sc[c * 2 + 1]};
          float mul[2] = {g[0].x * rscale, g[1].x * rscale};
          float add[2] = {g[0].z + off, g[1].z + off};
          if (edge) {
            // K's scales go in here, so that a hidden logit is -inf whatever its
            // group's scales are
            hide(v, hi - (k0 + c * 32), lo - (k0 + c * 32), g[0].x, g[1].x);
            mul[0] = mul[1] = rscale;
            if (dead >> (c * 2) & 1) add[0] = 0.f;
            if (dead >> (c * 2) & 2) add[1] = 0.f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2 s2;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 x = fma2(make_float2(__uint_as_float(v[h * 16 + 2 * k]),
                                                __uint_as_float(v[h * 16 + 2 * k + 1])),
                                    make_float2(mul[h], mul[h]), make_float2(add[h], add[h]));
              const float2 e = make_float2(ex2(x.x), ex2(x.y));
              s2 = k ? add2(s2, e) : e;
              pk[h * 8 + k] = pack_half2(e.x, e.y);
            }
            const float sum = s2.x + s2.y;
            if (sum != 0.f) l = fmaf(sum, g[h].w, l);
          }
          tmem_st16(s_col + c * 16, pk);
        };
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32];
          tmem_load(s_col + c * 32, v);
          probabilities(c, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + i);
      }
      // ---- the segment's rows
      wait(o_full + i, at - 1);
      __syncwarp();
      tc_fence_after();
      const bool whole = w.whole();
      const int slot = w.slot();
      *mine = l;
      named_barrier(1 + i, 256);
      l += *other;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int e_o = (int)e_v;                       // 2^E down to 2^-149; apart from inv: the product may leave fp32's range
      const float unit = exp2_int(e_o >> 1) * exp2_int(e_o - (e_o >> 1));
      if (whole) {
        // through the warp's own rows and half of the Q tile (its last MMA is
        // done), so that whole lines leave together
        uint8_t* stage = q_tile + (warp & 3) * 32 * 128;
        constexpr int kHalfLanes = D / 16;      // 16-byte chunks of half a row
        auto staged = [&](int wr, int ch) {     // chunk ch of the half
          const int c = half * kHalfLanes + ch;
          return reinterpret_cast<uint4*>(stage + ((c >> 3) * kTok + wr) * 128 + (((c & 7) ^ (wr & 7)) << 4));
        };
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t v[32];
          tmem_load(o_col + c * 32, v);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = pack_out(bf16, __uint_as_float(v[x * 8 + 2 * k]) * inv * unit,
                              __uint_as_float(v[x * 8 + 2 * k + 1]) * inv * unit);
            *staged(lane, c * 4 + x) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        __syncwarp();
#pragma unroll 2
        for (int c = 0; c < kHalfLanes; ++c) {
          const int wr = c * (32 / kHalfLanes) + lane / kHalfLanes, ch = lane % kHalfLanes;
          const int tr = (warp & 3) * 32 + wr;
          const uint4 v = *staged(wr, ch);
          if (i * 128 + tr < rows) {
            const int ur = row0 + tr, tk = p.token_of(ur);
            *reinterpret_cast<uint4*>((uint16_t*)p.out + ((int64_t)(w.u.q0 + tk) * p.heads + w.u.head * p.group +
                                                          ur - tk * p.group) * D + half * (D / 2) + ch * 8) = v;
          }
        }
      } else {
        // partials as shares of the row's mass: free of E and of the reference
        float4* part = p.part_o + ((int64_t)blockIdx.x * 2 + slot) * (D / 4) * kUnitRows + r;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t v[32];
          tmem_load(o_col + c * 32, v);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            part[(half * (D / 8) + c * 8 + x) * kUnitRows] =
                make_float4(__uint_as_float(v[4 * x]) * inv * unit, __uint_as_float(v[4 * x + 1]) * inv * unit,
                            __uint_as_float(v[4 * x + 2]) * inv * unit, __uint_as_float(v[4 * x + 3]) * inv * unit);
        }
      }
      const float lse2 = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + lg2(l) - kVLog;
      if (half == 0 && !whole) {
        p.part_lse[((int64_t)blockIdx.x * 2 + slot) * kUnitRows + r] = lse2;
      } else if (half == 0 && live && p.out_lse) {
        p.out_lse[(int64_t)(w.u.q0 + tok) * p.heads + w.u.head * p.group + urow - tok * p.group] = lse2 * kLn2;
      }
      if (threadIdx.x == 0 && !whole && w.skipped() == 0) {
        // the CTA with the unit's first tile names the merge, over the CTAs up to
        // the one whose range (start(c) = total c / ctas) holds its last tile
        MergeUnit mu;
        const int64_t total = misc[3], ctas = min((int64_t)gridDim.x, total);
        const int64_t u_end = quotient(total * blockIdx.x, ctas) + w.u_end();
        mu.parts = (int)quotient(u_end * ctas - 1, total) - (int)blockIdx.x + 1;
        mu.slot0 = slot;
        mu.q0 = w.u.q0;
        mu.row0 = w.u.rt * kUnitRows;
        mu.head = w.u.head;
        mu.rows = rows;
        *merge_s = mu;
      }
      tc_fence_before();
      named_barrier(1 + i, 256);    // both halves are done with the Q tile and the exchanged sums
    }
  }
  if (!ok) atomicOr(p.err, TKV_DEVERR_TIMEOUT);
  // every TMEM access and MMA of the CTA has completed
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0)
    p.merges[blockIdx.x] = *merge_s;
  if (warp == 20) {
    tc_fence_after();
    tmem_free(tmem, kManyTmem);
  }
}

// Joins the partial rows of a split unit: CTA (c, y) takes 8 elements of every
// row of the unit that starts in CTA c of many_rows_kernel and ends in a later
// one.  Latency bound: the parts' loads do not depend on one another, and are
// spread over as many CTAs as the row has 32-byte pieces (with 128-byte pieces,
// one part after the other, 21 us for a batch of drafted tokens; 9 us so), a trip
// to L2 for each kMergeParts parts (2 and 8 parts a trip take as long).
constexpr int kMergeCols = 8;
constexpr int kMergeParts = 4;
template <int D>
__global__ void __launch_bounds__(kUnitRows) merge_rows_kernel(const __grid_constant__ AttnParams8 p) {
  pdl_wait();
  const MergeUnit u = p.merges[blockIdx.x];
  const int r = threadIdx.x;
  if (u.parts == 0 || r >= u.rows) return;
  // part 0 sits in slot0 of CTA c, the others in slot 0 of theirs
  auto at = [&](int i) { return ((int64_t)(blockIdx.x + i) * 2 + (i ? 0 : u.slot0)); };
  float mx = -INFINITY, sum = 0.f;
  float o[kMergeCols] = {};
#pragma unroll 1
  for (int i = 0; i < u.parts; i += kMergeParts) {
    float lse[kMergeParts];
    float4 v[kMergeParts][kMergeCols / 4];
#pragma unroll
    for (int j = 0; j < kMergeParts; ++j) {   // past the last part: the last part again, dropped below
      const int64_t k = at(min(i + j, u.parts - 1));
      lse[j] = __ldcg(p.part_lse + k * kUnitRows + r);
      const float4* src = p.part_o + (k * (D / 4) + blockIdx.y * (kMergeCols / 4)) * kUnitRows + r;
#pragma unroll
      for (int x = 0; x < kMergeCols / 4; ++x) v[j][x] = __ldcg(src + x * kUnitRows);
    }
    float mn = mx;
#pragma unroll
    for (int j = 0; j < kMergeParts; ++j) mn = fmaxf(mn, lse[j]);
    const float back = mx == -INFINITY ? 0.f : ex2(mx - mn);
    mx = mn;
    sum *= back;
#pragma unroll
    for (int x = 0; x < kMergeCols; ++x) o[x] *= back;
#pragma unroll
    for (int j = 0; j < kMergeParts; ++j) {
      if (i + j >= u.parts) break;
      const float f = lse[j] == -INFINITY ? 0.f : ex2(lse[j] - mx);
      sum += f;
#pragma unroll
      for (int x = 0; x < kMergeCols / 4; ++x) {
        o[4 * x] += v[j][x].x * f;
        o[4 * x + 1] += v[j][x].y * f;
        o[4 * x + 2] += v[j][x].z * f;
        o[4 * x + 3] += v[j][x].w * f;
      }
    }
  }
  const int urow = u.row0 + r, tok = p.token_of(urow);
  const int64_t orow = (int64_t)(u.q0 + tok) * p.heads + u.head * p.group + urow - tok * p.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const bool bf16 = p.bf16 != 0;
  *reinterpret_cast<uint4*>((uint16_t*)p.out + orow * D + blockIdx.y * kMergeCols) =
      make_uint4(pack_out(bf16, o[0] * inv, o[1] * inv), pack_out(bf16, o[2] * inv, o[3] * inv),
                 pack_out(bf16, o[4] * inv, o[5] * inv), pack_out(bf16, o[6] * inv, o[7] * inv));
  if (blockIdx.y == 0 && p.out_lse) p.out_lse[orow] = sum == 0.f ? -INFINITY : (mx + lg2(sum)) * kLn2;
}

// ---------------------------------------------------------------- host side
size_t many_rows_scratch(int sms, int d) {
  return (size_t)sms * 2 * kUnitRows * (d + 1) * sizeof(float) + (size_t)sms * sizeof(MergeUnit) + 512;
}

namespace {
template <int D, int FMT>
cudaError_t launch_many(AttnParams8 p, const CUtensorMap* maps, int sms, cudaStream_t stream) {
  using L = ManyLayout<D>;
  uint8_t* at = p.data;
  p.part_o = reinterpret_cast<float4*>(at);
  at += (size_t)sms * 2 * kUnitRows * D * sizeof(float);
  p.part_lse = reinterpret_cast<float*>(at);
  at += (size_t)sms * 2 * kUnitRows * sizeof(float);
  p.merges = reinterpret_cast<MergeUnit*>(at);
  auto kern = many_rows_kernel<D, FMT>;
  static std::atomic<uint64_t> allowed;
  cudaError_t e = allow_smem(kern, L::kBytes, allowed);
  if (e != cudaSuccess) return e;
  e = launch_dependent(kern, dim3(sms), kManyThreads, L::kBytes, stream, p, maps[0], maps[1]);
  if (e != cudaSuccess) return e;
  return launch_dependent(merge_rows_kernel<D>, dim3(sms, D / kMergeCols), kUnitRows, 0, stream, p);
}
}  // namespace

cudaError_t launch_many_rows(const AttnParams8& p, const CUtensorMap* maps, int sms, int d, int format,
                             cudaStream_t stream) {
  if (d == 128)
    return format == TKV_KV8_INT8 ? launch_many<128, TKV_KV8_INT8>(p, maps, sms, stream)
                                  : launch_many<128, TKV_KV8_E4M3>(p, maps, sms, stream);
  return format == TKV_KV8_INT8 ? launch_many<64, TKV_KV8_INT8>(p, maps, sms, stream)
                                : launch_many<64, TKV_KV8_E4M3>(p, maps, sms, stream);
}

}  // namespace tkv
