// tkv_kv8_attn.cu -- attention over the 8-bit paged cache for requests with
// few query rows (single tokens, drafted tokens, short chunks).
//
// A row is one (query token, query head); the rows of a kv head share its K/V,
// so they are packed into tiles of 8 * NT rows (NT 1 or 2) and every code is read once per
// tile.  At few rows the kernel is bound by HBM: 2 head_dim bytes per token and
// kv head against 4 head_dim rows flops.  32 x 32768 tokens, 8 kv heads of 128:
// 389 us with int8 codes, 5.5 TB/s, whose expansion takes twice the
// instructions of e4m3's: 334 us, 6.4 TB/s (from a graph, in runs of some 10 ms;
// under the power limit of longer ones 416-442 and 360-373 us).
//
// Work is a flat list of steps -- 128 tokens (4 warps x 32) of one (request, kv
// head, row tile) unit, units in order -- cut into one contiguous range per
// resident CTA, so ragged batches and single long contexts load every SM
// alike; where there is little work, each CTA gets a part of one unit instead,
// so that none ends a unit twice.  A CTA that covers a whole unit writes the output; otherwise it
// leaves (max, sum, accumulator) partials in the workspace and the last CTA of
// the unit to arrive merges them in CTA order (the result does not depend on
// which one is last).
//
// Inside a CTA one warp produces: it walks the block table and fills a ring of
// stages (TMA boxes of K and V codes, scales by 4-byte asynchronous copies), ahead
// over unit boundaries.  Each of the four consumer warps takes 32 tokens of a
// stage, computes S^T = K Q^T and O^T += V^T P^T with mma.m16n8k16 on codes
// expanded to fp16 (exact for int8 and e4m3), and keeps its own softmax
// statistics; they meet only at the end of a unit.
//
// Scales: K's multiplies the logits in fp32.  V's is folded into P, normalised
// by a power of two (vinv) so that P stays in fp16's normal range for any
// scale; queries in bf16 become fp16 through a power of two per row, which
// only drops bits 2^-28 below the row's maximum.  P is rounded to fp16 (11 bits,
// 8 times finer than the bf16 of the usual fused kernels).  Where that would show
// beside the output's own rounding, with fp16 outputs, and the tile has idle
// columns, at up to 4 rows, those take what the rounding left over, and the two
// sums meet at the end of the unit: 22 bits without another MMA (error against 64
// bits of the 32 x 32768 tokens 0.0002, that of the output's rounding, instead of
// 0.0003; 389 us against 378 in short runs, the same under the power limit).  A
// second product for tiles of more rows took 22 % longer at 16 rows and was left
// out.  Sums, maxima and accumulators are fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

#include "tkv_kv8.h"
#include "tkv_kv8_common.cuh"
#include "tkv_ptx.cuh"

namespace tkv {

// Which kernel takes a request, by its rows per kv head.  When no request has
// more than 16, all run here, in row tiles of 8 or 16.  Otherwise requests of up
// to 8 rows run here and the others in many_rows_kernel, whose smallest tile of
// 128 rows still beats this kernel's 16-row instance for a batch of both (23
// requests of up to 9001 tokens with 28 rows each: 49 us against 56, with 35: 49
// against 78; chunks beside single tokens: 80 against 95), though not for 16 rows
// alone (32 requests of 4 tokens over 32768, 32 / 8 heads of 128: 577 us here
// against 1071, with e4m3 codes 476 against 1032).
// Small batches are the exception: up to 48 rows, and as long as the tables leave
// every CTA at most 32 steps, all run here, which saves the second kernel and the
// join (42 rows over 3000 tokens, 4 requests: 20 us against 31, 16 requests: 43
// against 48, 32 requests: 72 both; 64 rows, 4 requests: 53 against 42).
constexpr int kFewRowsAlone = 16;
constexpr int kFewRowsBeside = 8;
constexpr int kFewRowsShort = 48;
constexpr int kShortSteps = 32;
static int few_row_tiles(int64_t rows) { return rows <= 8 ? 1 : 2; }
constexpr int kFewCtasPerSm = 2;

constexpr int kFewWarps = 4;
constexpr int kFewConsumers = 32 * kFewWarps;
constexpr int kFewThreads = kFewConsumers + 32;       // and the producer warp
constexpr int kTileTok = 32;                          // tokens of a warp's tile
constexpr int kStepTok = kTileTok * kFewWarps;        // tokens of a step
// What ending one unit and starting the next costs a CTA, in steps: up to this
// many more steps than an even share, each CTA takes a part of one unit only
// (4 requests of 2048 tokens: 11.7 us against 14.4; drafted tokens 45 against
// 50; a 131071-token context the same; with up to 16 steps more, 16 requests of
// 2048 tokens take 31 us against 24).
constexpr int kBoundarySteps = 2;
// Parts of a unit that one trip to L2 fetches when they are joined, maxima and
// accumulators together (a 131071-token context, 36 parts: 52.7 us; a first trip
// for all maxima and then 8 accumulators a trip: 56.6).
constexpr int kJoin = 12;

template <int D, int NT>
struct FewLayout {
  static constexpr int kStages = D == 64 ? 5 : 3;      // what two CTAs an SM have room for
  static constexpr int kRows = 8 * NT;
  static constexpr int kHalf = kStepTok * D;           // codes of K (or V) in a stage
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kStages * kStage;
  // fp16 queries, rows D + 16 apart (8-byte fragment reads of 4 rows hit 32
  // banks), and the accumulators that the warps add up at the end of a unit;
  // with the query fragments in registers the two share their space
  static constexpr bool kQRegs = NT == 1;
  static constexpr int kQStride = D + 16;
  static constexpr int kMergeStride = D + 4;
  static constexpr int kQBytes = kRows * kQStride * 2;
  static constexpr int kMergeBufs = NT == 1 ? 2 : 1;
  static constexpr int kMergeBytes = kMergeBufs * kRows * kMergeStride * 4;
  static constexpr int kQOff = kRing;
  static constexpr int kMergeOff = kQRegs ? kQOff : kQOff + kQBytes;
  static constexpr int kStatOff = kMergeOff + (kMergeBytes > kQBytes ? kMergeBytes : kQBytes);  // [warps][rows][2], row scales
  static constexpr int kScaleOff = kStatOff + (kFewWarps + 1) * kRows * 8;   // [stages][16]: K's, V's
  static constexpr int kBarOff = kScaleOff + kStages * 64;
  static constexpr int kMiscOff = kBarOff + kStages * 16;
  static constexpr int kBytes = kMiscOff + 88;
};

// Where a walk over the units stands.
struct UnitPos {
  int req;        // request
  int head;       // kv head
  int rt;         // row tile
  int q0, q_len;  // first packed token, query tokens
  int kv;         // keys
  int tiles_r;    // row tiles of the request
  int step0;      // first step (of 128 tokens) of the request's units
  int steps;      // steps of each of its units
};

template <int RT>
__device__ __forceinline__ bool load_request(const AttnParams8& p, int bs, int req, UnitPos& u) {
  u.req = req;
  const RequestLens n = request_lens(p, bs, req);
  u.q0 = n.q0;
  u.q_len = n.q_len;
  u.kv = n.kv;
  if (!n.few_rows(p)) {
    u.steps = 0;
    u.tiles_r = 0;
    return false;
  }
  u.tiles_r = (n.q_len * p.group + RT - 1) / RT;
  const int lo = n.first_key(p);
  u.step0 = lo / kStepTok;
  // a request without keys keeps one empty step, which writes its zeros
  u.steps = max(1, (n.kv + kStepTok - 1) / kStepTok - u.step0);
  return u.tiles_r > 0;
}

// Places of a request in the list that the CTAs share: its steps (chunk 0), or
// its parts of up to `chunk` steps.
template <int RT>
__device__ __forceinline__ int64_t request_places(const AttnParams8& p, int bs, int req, int chunk, int64_t& units) {
  UnitPos u;
  if (!load_request<RT>(p, bs, req, u)) return 0;
  const int64_t n = (int64_t)u.tiles_r * p.kv_heads;
  units += n;
  return n * (chunk ? (u.steps + chunk - 1) / chunk : u.steps);
}

// Next unit in order; false past the last request.
template <int RT>
__device__ __forceinline__ bool next_unit(const AttnParams8& p, int bs, UnitPos& u) {
  if (++u.rt < u.tiles_r) return true;
  u.rt = 0;
  if (++u.head < p.kv_heads) return true;
  u.head = 0;
  for (int r = u.req + 1; r < p.requests; ++r)
    if (load_request<RT>(p, bs, r, u)) return true;
  return false;
}

template <int D, int BOXES, int FMT, int NT>
__global__ void __launch_bounds__(kFewThreads, kFewCtasPerSm)
    few_rows_kernel(const __grid_constant__ AttnParams8 p, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v) {
  using L = FewLayout<D, NT>;
  constexpr int RT = L::kRows;
  constexpr int S = L::kStages;
  constexpr int kBoxes = BOXES;                         // TMA boxes of a warp's tile (K; V alike)
  constexpr int kBox = kTileTok / kBoxes;               // rows of a box
  constexpr int kStepBoxes = kFewWarps * kBoxes;        // boxes of a step (K; V alike)
  const int bs = p.block_size;
  const bool bf16 = p.bf16 != 0;
  constexpr int kBatch = 32 / kStepBoxes;               // steps whose table cells the producer holds
  constexpr int kSwz = D == 128 ? 7 : 3;
  extern __shared__ __align__(1024) uint8_t few_smem[];
  uint8_t* smem = few_smem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  __half* q_s = reinterpret_cast<__half*>(smem + L::kQOff);
  float* merge_s = reinterpret_cast<float*>(smem + L::kMergeOff);
  float* stat_s = reinterpret_cast<float*>(smem + L::kStatOff);
  float* rscale_s = stat_s + kFewWarps * RT * 2;         // [RT] logit scale of each row
  float* scale_s = reinterpret_cast<float*>(smem + L::kScaleOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + S;
  int64_t* range_s = reinterpret_cast<int64_t*>(smem + L::kMiscOff);   // [5] scan scratch
  int64_t* units_s = range_s + 5;                                       // [5]
  int* flag_s = reinterpret_cast<int*>(smem + L::kMiscOff + 80);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full + s, 1 + 2 * kStepBoxes);   // one expect_tx arrival and one per scale-copying lane
      mbar_init(empty + s, kFewWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }

  pdl_launch_dependents();
  pdl_wait();   // everything below reads what the kernels before may have written

  // ---- this CTA's range of the flat step list, or its part of one unit
  UnitPos unit;
  int64_t total, ctas, begin, end, unit_at;   // unit_at: flat index of the unit's first step
  int chunk = 0;                              // steps of a part, 0: ranges over unit boundaries
  int part0 = 0, parts0 = 0;                  // first CTA and count of the unit's parts
  {
    const int per = (p.requests + kFewThreads - 1) / kFewThreads;
    const int r0 = min(p.requests, (int)threadIdx.x * per), r1 = min(p.requests, r0 + per);
    int64_t at, mine;                         // first place and places of this thread's requests
    auto scan = [&](int64_t& units) {
      mine = 0;
      for (int r = r0; r < r1; ++r) mine += request_places<RT>(p, bs, r, chunk, units);
      int64_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += x;
      }
      units = warp_sum(units);
      if (lane == 31) {
        range_s[warp] = inc;
        units_s[warp] = units;
      }
      __syncthreads();
      at = inc - mine;
      total = units = 0;
#pragma unroll
      for (int w = 0; w < kFewThreads / 32; ++w) {
        if (w < warp) at += range_s[w];
        total += range_s[w];
        units += units_s[w];
      }
      __syncthreads();
    };
    int64_t units = 0;
    scan(units);
    const int64_t grid = gridDim.x;
    if (units < grid) {
      const int64_t c = quotient(total + grid - units - 1, grid - units);
      if (c * grid <= total + kBoundarySteps * grid) {
        chunk = (int)c;                       // total / c + units parts at most
        scan(units);
      }
    }
    ctas = min(grid, total);                  // every range holds a place
    if (blockIdx.x >= ctas) return;
    begin = chunk ? blockIdx.x : quotient(total * blockIdx.x, ctas);
    end = chunk ? 0 : quotient(total * (blockIdx.x + 1), ctas);
    if (at <= begin && begin < at + mine) {
      int r = r0;
      for (;; ++r) {
        const int64_t n = request_places<RT>(p, bs, r, chunk, units);
        if (begin < at + n) break;
        at += n;
      }
      range_s[0] = at;
      range_s[1] = r;
    }
    __syncthreads();
    load_request<RT>(p, bs, (int)range_s[1], unit);
    int in;                                   // unit of the request
    if (chunk) {
      const int place = (int)(begin - range_s[0]);
      parts0 = (unit.steps + chunk - 1) / chunk;
      in = place / parts0;
      part0 = blockIdx.x - (place - in * parts0);
      begin = (int64_t)(place - in * parts0) * chunk;
      end = min(begin + chunk, (int64_t)unit.steps);
      unit_at = 0;
    } else {
      in = (int)quotient(begin - range_s[0], unit.steps);
      unit_at = range_s[0] + (int64_t)in * unit.steps;
    }
    unit.head = in / unit.tiles_r;
    unit.rt = in - unit.head * unit.tiles_r;
  }

  bool ok = true;
  if (warp == kFewWarps) {
    // ---- producer: lane = box of the step (K in [0, kStepBoxes), V in [kStepBoxes, 2 kStepBoxes))
    const int box = lane % kStepBoxes;
    const bool is_v = lane >= kStepBoxes;
    const CUtensorMap* map = is_v ? &tm_v : &tm_k;
    const float* scales = is_v ? p.v_scale : p.k_scale;
    const uint32_t code_off = (is_v ? L::kHalf : 0) + box * kBox * D;
    int32_t cells = 0;                    // table cell of box lane % kStepBoxes, step lane / kStepBoxes of the batch
    int left = 0;                         // steps left in the batch
    int64_t issued = 0;
    for (int64_t at = begin; at < end; ++at, ++issued) {
      if (at >= unit_at + unit.steps) {
        unit_at += unit.steps;
        next_unit<RT>(p, bs, unit);
        left = 0;
      }
      const int step = unit.step0 + (int)(at - unit_at);
      if (left == 0) {
        left = kBatch;
        const int tok = (step + lane / kStepBoxes) * kStepTok + box * kBox;
        cells = tok < unit.kv ? p.table[unit.req * p.table_stride + tok / bs] : -1;
      }
      const int cell = __shfl_sync(~0u, cells, (kBatch - left) * kStepBoxes + box);
      --left;
      const int tok = step * kStepTok + box * kBox;
      const int any_lo = p.window > 0 ? unit.kv - unit.q_len - p.window + 1 : 0;
      const bool in_keys = tok < unit.kv && tok + kBox > any_lo && lane < 2 * kStepBoxes;
      const bool good = in_keys && cell >= 0 && cell < p.blocks;
      const int s = (int)(issued % S);
      // one lane's timeout is the warp's: the votes below want all of it
      if (!__all_sync(~0u, mbar_wait(empty + s, (uint32_t)((issued / S) & 1) ^ 1))) {
        ok = false;
        break;
      }
      const uint32_t bytes = __popc(__ballot_sync(~0u, in_keys)) * kBox * D;
      // zero scales are plain stores, which lane 0's arrival (a release, unlike
      // those of the asynchronous copies) makes visible to the consumers
      float* dst = scale_s + s * 16 + lane;
      if (lane < 2 * kStepBoxes && !good) *dst = 0.f;
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(full + s, bytes);
      __syncwarp();
      if (lane < 2 * kStepBoxes) {
        if (in_keys) {
          // a bad slot's box lies before the cache, which TMA fills with zeros
          tma_load_2d(smem + s * L::kStage + code_off, map, 0,
                      good ? (cell * p.kv_heads + unit.head) * bs + (tok & (bs - 1)) : -kBox, full + s);
          if (!good) atomicOr(p.err, TKV_DEVERR_BAD_SLOT);
        }
        if (good) cp_async4(dst, scales + (int64_t)cell * p.kv_heads + unit.head);
        cp_async_mbar_arrive(full + s);
      }
    }
    // no copy may still be landing when the CTA exits
    for (int64_t i = max((int64_t)0, issued - S); i < issued; ++i)
      ok = mbar_wait(full + i % S, (uint32_t)((i / S) & 1)) && ok;
    if (!ok && lane == 0) atomicOr(p.err, TKV_DEVERR_TIMEOUT);
    return;                               // the consumers' barriers do not count this warp
  }

  // ---- units
  const int lm_row = (lane & 7) + ((lane >> 3) & 1) * 8;   // ldmatrix: row and 16-byte chunk of this lane
  const int lm_chunk = lane >> 4;
  int64_t consumed = 0;
  int64_t pos = begin;
  while (pos < end) {
    const int64_t seg_end = min(end, unit_at + unit.steps);
    const int rows = min(RT, unit.q_len * p.group - unit.rt * RT);
    const int nact = (rows + 7) / 8;
    const int row0 = unit.rt * RT;       // first row of the tile within the request
    // Up to 4 rows leave half of the tile's columns idle: columns 4-7 repeat rows
    // 0-3, and take what the rounding of P to fp16 leaves over in columns 0-3.
    const bool twin = NT == 1 && !bf16 && rows <= 4;
    const float rest = t4 >= 2 ? -1.f : 0.f;
    const auto row_of = [&](int r) { return twin ? r & 3 : r; };
    // the rows' queries as fp16, and their logit scales
    for (int r = warp; r < RT; r += kFewWarps) {
      constexpr int E = D / 64;            // words per lane
      float2 x[E];
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = make_float2(0.f, 0.f);
      if (row_of(r) < rows) {
        const int row = row0 + row_of(r);
        const int tok = unit.q0 + row / p.group, h = unit.head * p.group + row % p.group;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(
            (const uint16_t*)p.q.data + tok * p.q.token_stride + h * p.q.head_stride);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[i] = unpack_in(bf16, src[lane + 32 * i]);
          amax = fmaxf(amax, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
        }
      }
      float up = 1.f, down = 1.f;
      if (bf16) fp16_scale(warp_max(amax), up, down);
#pragma unroll
      for (int i = 0; i < E; ++i)
        *reinterpret_cast<uint32_t*>(q_s + r * L::kQStride + 2 * (lane + 32 * i)) =
            pack_half2(x[i].x * up, x[i].y * up);
      if (lane == 0) rscale_s[r] = p.scale_log2 * down;
    }
    named_barrier(1, kFewConsumers);
    constexpr bool kQRegs = L::kQRegs;
    uint2 qf[kQRegs ? NT : 1][kQRegs ? D / 16 : 1];
    if constexpr (kQRegs) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          qf[n][c] = *reinterpret_cast<const uint2*>(q_s + (n * 8 + g) * L::kQStride + c * 16 + 4 * t4);
    }
    float rs[NT][2];
    int limit[NT][2];                     // keys below limit are visible (and at or above limit - window)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = n * 8 + 2 * t4 + c;
        rs[n][c] = rscale_s[r];
        limit[n][c] = unit.kv - unit.q_len + (row0 + min(row_of(r), rows - 1)) / p.group + 1;
      }
    // every row sees keys [all_lo, all_hi)
    const int all_hi = unit.kv - unit.q_len + row0 / p.group + 1;
    const int all_lo = p.window > 0 ? unit.kv - unit.q_len + (row0 + rows - 1) / p.group + 1 - p.window : 0;
    const int any_lo = p.window > 0 ? unit.kv - unit.q_len - p.window + 1 : 0;

    float m[NT][2], l[NT][2], acc[NT][D / 16][4];
    float vinv = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int u = 0; u < D / 16; ++u) acc[n][u][0] = acc[n][u][1] = acc[n][u][2] = acc[n][u][3] = 0.f;
    }

#pragma unroll 1
    for (; pos < seg_end; ++pos) {
      const int s = (int)(consumed % S);
      if (ok && !mbar_wait(full + s, (uint32_t)((consumed / S) & 1))) {
        ok = false;
        if (lane == 0) atomicOr(p.err, TKV_DEVERR_TIMEOUT);
      }
      __syncwarp();
      const uint32_t tok_ = wait_token();
      const int tok0 = (unit.step0 + (int)(pos - unit_at)) * kStepTok + warp * kTileTok;
      uint8_t* st = smem + s * L::kStage + warp * (kTileTok * D);
      if (tok0 < unit.kv && tok0 + kTileTok > any_lo) {
        const uint32_t kaddr = after(smem_u32(st), tok_);
        const bool edge = tok0 + kTileTok > all_hi || tok0 < all_lo;
        if (tok0 + kTileTok > unit.kv || tok0 < any_lo) {
          // rows nobody sees may hold anything: their values must not reach the MMA
          for (int i = lane; i < kTileTok * D / 16; i += 32) {
            const int tk = tok0 + i / (D / 16);
            if (tk >= unit.kv || tk < any_lo) *reinterpret_cast<uint4*>(st + L::kHalf + i * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();   // the stage's next TMA write comes after these stores
          __syncwarp();
        }
        const uint32_t vaddr = after(kaddr + L::kHalf, wait_token());
        float ks[kBoxes], vs[kBoxes];
#pragma unroll
        for (int b = 0; b < kBoxes; ++b) {
          ks[b] = scale_s[s * 16 + warp * kBoxes + b];
          vs[b] = scale_s[s * 16 + kStepBoxes + warp * kBoxes + b];
        }
        // S^T: 2 x 16 tokens, 8 NT rows
        float sc[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) sc[n][h][0] = sc[n][h][1] = sc[n][h][2] = sc[n][h][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t off = (uint32_t)((h * 16 + lm_row) * D + (c + lm_chunk) * 16);
            ldsm_x4(kaddr + swz<kSwz>(off), a[h][0], a[h][1], a[h][2], a[h][3]);
          }
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t f[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              expand4<FMT>(a[h][2 * cc], f[h][0], f[h][2]);
              expand4<FMT>(a[h][2 * cc + 1], f[h][1], f[h][3]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (n < nact) {
                uint2 b;
                if constexpr (kQRegs) b = qf[n][c + cc];
                else b = *reinterpret_cast<const uint2*>(q_s + (n * 8 + g) * L::kQStride + (c + cc) * 16 + 4 * t4);
                mma_16816(sc[n][0], f[0][0], f[0][1], f[0][2], f[0][3], b.x, b.y);
                mma_16816(sc[n][1], f[1][0], f[1][1], f[1][2], f[1][3], b.x, b.y);
              }
          }
        }
        // V's scale relative to the power of two the accumulators carry
        float vn[kBoxes];
#pragma unroll
        for (int b = 0; b < kBoxes; ++b) {
          if (vs[b] > 0.f && vs[b] < 3e38f && (vinv == 0.f || vs[b] * vinv > 32768.f)) {
            const float nv = scale_inverse(vs[b]);
            const float r = vinv == 0.f ? 0.f : nv / vinv;
            vinv = nv;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int u = 0; u < D / 16; ++u)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[n][u][x] *= r;
          }
        }
#pragma unroll
        for (int b = 0; b < kBoxes; ++b) vn[b] = vs[b] * vinv;
        uint32_t pb[NT][2][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n >= nact) continue;
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int c = x & 1;
              float v = sc[n][h][x] * (ks[h * kBoxes / 2] * rs[n][c]);
              if (edge) {
                const int tk = tok0 + h * 16 + g + (x >> 1) * 8;
                if (tk >= limit[n][c] || (p.window > 0 && tk < limit[n][c] - p.window)) v = -INFINITY;
              }
              sc[n][h][x] = v;
              mx[c] = fmaxf(mx[c], v);
            }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(~0u, mx[0], o));
            mx[1] = fmaxf(mx[1], __shfl_xor_sync(~0u, mx[1], o));
          }
          if (__any_sync(~0u, mx[0] > m[n][0] || mx[1] > m[n][1])) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float mn = fmaxf(m[n][c], mx[c]);
              const float r = mn == -INFINITY ? 1.f : ex2(m[n][c] - mn);
              m[n][c] = mn;
              l[n][c] *= r;
#pragma unroll
              for (int u = 0; u < D / 16; ++u) {
                acc[n][u][c] *= r;
                acc[n][u][2 + c] *= r;
              }
            }
          }
          const float base[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float w = ex2(sc[n][h][x] - base[x & 1]);
              l[n][x & 1] += w;
              e[x] = w * vn[h * kBoxes / 2];
              if (edge && sc[n][h][x] == -INFINITY) e[x] = 0.f;   // also under a NaN scale
            }
            uint32_t p0 = pack_half2(e[0], e[1]), p1 = pack_half2(e[2], e[3]);
            if (twin) {
              const float2 r0 = unpack_in(false, p0), r1 = unpack_in(false, p1);
              p0 = pack_half2(fmaf(rest, r0.x, e[0]), fmaf(rest, r0.y, e[1]));
              p1 = pack_half2(fmaf(rest, r1.x, e[2]), fmaf(rest, r1.y, e[3]));
            }
            pb[n][h][0] = movmatrix_t(p0);
            pb[n][h][1] = movmatrix_t(p1);
          }
        }
        // O^T += V^T P^T: lane (g, t4) owns head_dim elements [g D / 8, (g + 1) D / 8)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr int W = D / 32;   // words of codes per token and lane
          uint32_t w[4][W];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tk = h * 16 + 2 * t4 + (i & 1) + (i >> 1) * 8;
            const uint32_t ad = vaddr + swz<kSwz>((uint32_t)(tk * D + g * (D / 8)));
            if constexpr (W == 4) {
              const uint4 v = lds128(ad);
              w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
            } else {
              const uint2 v = lds64(ad);
              w[i][0] = v.x, w[i][1] = v.y;
            }
          }
#pragma unroll
          for (int j = 0; j < W; ++j) {
            uint32_t a0[4], a1[4];   // tokens (2t, 2t+1), (2t+8, 2t+9) of elements 4j .. 4j+3
            expand_pairs<FMT>(w[0][j], w[1][j], a0);
            expand_pairs<FMT>(w[2][j], w[3][j], a1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (n < nact) {
                mma_16816(acc[n][2 * j], a0[0], a0[1], a1[0], a1[1], pb[n][h][0], pb[n][h][1]);
                mma_16816(acc[n][2 * j + 1], a0[2], a0[3], a1[2], a1[3], pb[n][h][0], pb[n][h][1]);
              }
          }
        }
      }
      // the fragments' loads come before the stage's reuse: every one of them
      // feeds the first row tile's accumulators
#pragma unroll
      for (int u = 0; u < D / 16; ++u) hold(acc[0][u][0]);
      ++consumed;
      __syncwarp();   // every lane has read the stage
      if (lane == 0) mbar_arrive(empty + s);
    }

    // ---- the CTA's share of the unit: merge the warps' statistics and accumulators
    if (twin) {
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[0][u][x] += __shfl_xor_sync(~0u, acc[0][u][x], 2);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(~0u, l[n][c], o);
        if (g == 0) {
          stat_s[(warp * RT + n * 8 + 2 * t4 + c) * 2] = m[n][c];
          stat_s[(warp * RT + n * 8 + 2 * t4 + c) * 2 + 1] = l[n][c];
        }
      }
    named_barrier(1, kFewConsumers);
    float mm[NT][2], ll[NT][2];
    const float back = vinv == 0.f ? 0.f : 1.f / vinv;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = n * 8 + 2 * t4 + c;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) mx = fmaxf(mx, stat_s[(w * RT + r) * 2]);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          const float mw = stat_s[(w * RT + r) * 2], lw = stat_s[(w * RT + r) * 2 + 1];
          sum += mx == -INFINITY ? lw : lw * ex2(mw - mx);   // no key seen: 0, or NaN logits' sum
        }
        mm[n][c] = mx;
        ll[n][c] = sum;
        const float f = back * (mx == -INFINITY ? 1.f : ex2(m[n][c] - mx));
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
          acc[n][u][c] *= f;
          acc[n][u][2 + c] *= f;
        }
      }
    // warps 3 and 2 hand their accumulators to 1 and 0, then 1 to 0; with one
    // buffer 3 to 2, 1 to 0, 2 to 0
    auto put = [&](float* dst) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (n < nact)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* d = dst + (n * 8 + 2 * t4 + c) * L::kMergeStride + g * (D / 8);
#pragma unroll
            for (int u = 0; u < D / 16; u += 2)
              *reinterpret_cast<float4*>(d + 2 * u) =
                  make_float4(acc[n][u][c], acc[n][u][2 + c], acc[n][u + 1][c], acc[n][u + 1][2 + c]);
          }
    };
    auto add = [&](const float* src) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (n < nact)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float* d = src + (n * 8 + 2 * t4 + c) * L::kMergeStride + g * (D / 8);
#pragma unroll
            for (int u = 0; u < D / 16; u += 2) {
              const float4 v = *reinterpret_cast<const float4*>(d + 2 * u);
              acc[n][u][c] += v.x;
              acc[n][u][2 + c] += v.y;
              acc[n][u + 1][c] += v.z;
              acc[n][u + 1][2 + c] += v.w;
            }
          }
    };
    if constexpr (L::kMergeBufs == 2) {
      float* buf = merge_s + (warp & 1) * RT * L::kMergeStride;
      if (warp >= 2) put(buf);
      named_barrier(1, kFewConsumers);
      if (warp < 2) add(buf);
      __syncwarp();
      if (warp == 1) put(buf);
      named_barrier(1, kFewConsumers);
      if (warp == 0) add(merge_s + RT * L::kMergeStride);
    } else {
      for (int round = 0; round < 3; ++round) {
        const int from = round == 0 ? 3 : round == 1 ? 1 : 2, to = round == 0 ? 2 : 0;
        if (warp == from) put(merge_s);
        named_barrier(1, kFewConsumers);
        if (warp == to) add(merge_s);
        named_barrier(1, kFewConsumers);
      }
    }
    const int64_t u0 = unit_at, u1 = unit_at + unit.steps;
    const bool whole = begin <= u0 && end >= u1;
    const int slot = begin >= u0 ? 0 : 1;
    float* part = reinterpret_cast<float*>(p.data) + ((int64_t)blockIdx.x * 2 + slot) * RT * (D + 2);
    if (warp == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = n * 8 + 2 * t4 + c;
          if (r >= rows) continue;
          if (whole) {
            const float sum = ll[n][c], inv = sum == 0.f ? 0.f : 1.f / sum;
            const int64_t orow = (int64_t)(unit.q0 + (row0 + r) / p.group) * p.heads + unit.head * p.group +
                                 (row0 + r) % p.group;
            uint16_t* o = (uint16_t*)p.out + orow * D + g * (D / 8);
#pragma unroll
            for (int u = 0; u < D / 16; u += 4) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                w[x] = pack_out(bf16, acc[n][u + x][c] * inv, acc[n][u + x][2 + c] * inv);
              *reinterpret_cast<uint4*>(o + 2 * u) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (g == 0 && p.out_lse) p.out_lse[orow] = sum == 0.f ? -INFINITY : row_lse(mm[n][c], sum);
          } else {
            float* d = part + r * D + g * (D / 8);
#pragma unroll
            for (int u = 0; u < D / 16; u += 2)
              *reinterpret_cast<float4*>(d + 2 * u) =
                  make_float4(acc[n][u][c], acc[n][u][2 + c], acc[n][u + 1][c], acc[n][u + 1][2 + c]);
            if (g == 0) *reinterpret_cast<float2*>(part + RT * D + r * 2) = make_float2(mm[n][c], ll[n][c]);
          }
        }
    }
    if (!whole) {
      // CTAs whose ranges meet this unit: start(c) = total c / ctas
      const int c0 = chunk ? part0 : (int)quotient((u0 + 1) * ctas - 1, total);
      const int c1 = chunk ? part0 + parts0 - 1 : (int)quotient(u1 * ctas - 1, total);
      named_barrier(1, kFewConsumers);
      if (threadIdx.x == 0) {
        const uint32_t n = atom_add_acq_rel_gpu(p.counters + c0, 1u);
        *flag_s = n == (uint32_t)(c1 - c0);
        if (*flag_s) p.counters[c0] = 0;
      }
      named_barrier(1, kFewConsumers);
      if (*flag_s) {
        const int64_t stride = (int64_t)2 * RT * (D + 2);
        // CTA c0's share sits in slot 0 when its range starts at the unit, else in slot 1
        const float* first = reinterpret_cast<const float*>(p.data) +
                             ((int64_t)c0 * 2 + (chunk || quotient(total * c0, ctas) >= u0 ? 0 : 1)) * RT * (D + 2);
        const float* rest = reinterpret_cast<const float*>(p.data) + (int64_t)c0 * stride;
        const int parts = c1 - c0 + 1;
        constexpr int kLanes = D / 4;    // threads of a row
        for (int r = threadIdx.x / kLanes; r < rows; r += kFewConsumers / kLanes) {
          const int d4 = (threadIdx.x % kLanes) * 4;
          float mx = -INFINITY, sum = 0.f, o0 = 0.f, o1 = 0.f, o2 = 0.f, o3 = 0.f;
#pragma unroll 1
          for (int i = 0; i < parts; i += kJoin) {
            float2 ml[kJoin];
            float4 v[kJoin];
#pragma unroll
            for (int j = 0; j < kJoin; ++j) {
              ml[j] = make_float2(-INFINITY, 0.f);
              v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (i + j < parts) {
                const float* src = i + j ? rest + (i + j) * stride : first;
                ml[j] = __ldcg(reinterpret_cast<const float2*>(src + RT * D + r * 2));
                v[j] = __ldcg(reinterpret_cast<const float4*>(src + r * D + d4));
              }
            }
            float mn = mx;
#pragma unroll
            for (int j = 0; j < kJoin; ++j) mn = fmaxf(mn, ml[j].x);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float back = mx == -INFINITY && mn == -INFINITY ? 1.f : ex2(mx - base);
            mx = mn;
            sum *= back, o0 *= back, o1 *= back, o2 *= back, o3 *= back;
#pragma unroll
            for (int j = 0; j < kJoin; ++j) {
              const float f = mx == -INFINITY ? 1.f : ex2(ml[j].x - base);
              sum += ml[j].y * f;
              o0 += v[j].x * f, o1 += v[j].y * f, o2 += v[j].z * f, o3 += v[j].w * f;
            }
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int64_t orow = (int64_t)(unit.q0 + (row0 + r) / p.group) * p.heads + unit.head * p.group +
                               (row0 + r) % p.group;
          *reinterpret_cast<uint2*>((uint16_t*)p.out + orow * D + d4) =
              make_uint2(pack_out(bf16, o0 * inv, o1 * inv), pack_out(bf16, o2 * inv, o3 * inv));
          if (d4 == 0 && p.out_lse) p.out_lse[orow] = sum == 0.f ? -INFINITY : row_lse(mx, sum);
        }
      }
    }
    named_barrier(1, kFewConsumers);   // the shared buffers are free for the next unit
    if (pos < end) {
      unit_at += unit.steps;
      next_unit<RT>(p, bs, unit);
    }
  }
}

// ---------------------------------------------------------------- host side
static bool has_many_rows(const AttnParams8& p, int sms) {
  const int64_t rows = (int64_t)p.group * p.max_q_len;
  if (rows <= kFewRowsAlone) return false;
  if (rows > kFewRowsShort) return true;
  // what the step may hold at most: its row tiles, and the keys that a table has
  // room for or a window leaves
  const int64_t tiles = std::min<int64_t>(p.requests * ((rows + 15) / 16),
                                          (int64_t)p.tokens * p.group / 16 + p.requests);
  int64_t keys = (int64_t)p.table_width * p.block_size;
  if (p.window > 0) keys = std::min<int64_t>(keys, (int64_t)p.window + p.max_q_len + kStepTok);
  const int64_t steps = tiles * p.kv_heads * ((keys + kStepTok - 1) / kStepTok);
  return steps > (int64_t)kShortSteps * sms * kFewCtasPerSm;
}

namespace {

template <int D, int BOXES, int FMT, int NT>
cudaError_t launch_few(const AttnParams8& p, const CUtensorMap* maps, int sms, cudaStream_t stream) {
  using L = FewLayout<D, NT>;
  auto kern = few_rows_kernel<D, BOXES, FMT, NT>;
  static std::atomic<uint64_t> allowed;
  const cudaError_t e = allow_smem(kern, L::kBytes, allowed);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(sms * kFewCtasPerSm), kFewThreads, L::kBytes, stream, p, maps[0], maps[1]);
}

template <int D, int BOXES, int FMT>
cudaError_t few_nt(const AttnParams8& p, const CUtensorMap* maps, int sms, cudaStream_t s) {
  const int64_t rows = std::min<int64_t>((int64_t)p.group * p.max_q_len, p.few_rows_max);
  return few_row_tiles(rows) == 1 ? launch_few<D, BOXES, FMT, 1>(p, maps, sms, s)
                                  : launch_few<D, BOXES, FMT, 2>(p, maps, sms, s);
}

template <int D>
cudaError_t few_format(const AttnParams8& p, const CUtensorMap* maps, int sms, int format, cudaStream_t s) {
  if (p.block_size == 16)
    return format == TKV_KV8_INT8 ? few_nt<D, 2, TKV_KV8_INT8>(p, maps, sms, s)
                                  : few_nt<D, 2, TKV_KV8_E4M3>(p, maps, sms, s);
  return format == TKV_KV8_INT8 ? few_nt<D, 1, TKV_KV8_INT8>(p, maps, sms, s)
                                : few_nt<D, 1, TKV_KV8_E4M3>(p, maps, sms, s);
}

}  // namespace

void kv8_attention_scratch(int sms, int d, int group, int max_q_len, size_t* counters, size_t* data) {
  const int64_t rows = (int64_t)group * max_q_len;
  const int nt = few_row_tiles(rows);
  const size_t ctas = (size_t)sms * kFewCtasPerSm;
  *counters = ctas * sizeof(uint32_t);
  *data = ctas * 2 * 8 * nt * (d + 2) * sizeof(float);
  if (rows > kFewRowsAlone) *data = std::max(*data, many_rows_scratch(sms, d));
}

cudaError_t launch_kv8_attention(const AttnParams8& args, int sms, int d, int format, cudaStream_t stream) {
  AttnParams8 p = args;
  const bool many = has_many_rows(p, sms);
  // a lone request needs one kernel: the one for its largest possible size; and
  // without a request that max_q_len calls long, this kernel takes all
  p.few_rows_max = !many ? 0x7fffffff : p.requests == 1 ? 0 : kFewRowsBeside;
  CUtensorMap maps[2];
  if (!kv8_code_maps(p, d, maps)) return cudaErrorInvalidValue;
  if (p.few_rows_max > 0) {
    const cudaError_t e = d == 128 ? few_format<128>(p, maps, sms, format, stream)
                                   : few_format<64>(p, maps, sms, format, stream);
    if (e != cudaSuccess || !many) return e;
  }
  return launch_many_rows(p, maps, sms, d, format, stream);
}

}  // namespace tkv
