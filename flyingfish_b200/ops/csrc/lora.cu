// Low-rank adapters of many requests beside a shared projection:  Y[M,N] = X W^T + delta,  delta_r = B_a (s_a A_a x_r)  for the
// adapter a = ids[r] of row r, no delta where ids[r] is negative. A stack holds the adapters of one projection: A [adapters, R, K],
// B [adapters, N, R], scales (of an adapter, or of each of its rank rows) and ranks (rank rows behind an adapter's own are zero and not read). R is a multiple of 16.
//
//   lora_shrink_kernel (here)   t_r = s_a A_a x_r: [M, 2R], every value as two BF16 words, t = high + low
//   the product with W          gemm_skinny.cu, gemm_bf16.cu: B_a t_r is accumulated behind the product's own K blocks (lora.cuh), one rounding at the end
//
// t in two BF16 words: the second product's tensor instructions take BF16; one word would leave 2^-9 of t, two leave 2^-17 or less.
//
// The shrink is bound by its bytes: X once, and A of the adapters in use. The order of its sums depends on K alone.
#include "lora.cuh"
#include "launchers.h"

namespace ff {

constexpr int LS_SPLIT = 8;          // CTAs of a cluster share K
constexpr int LS_ROWS = 128;         // rows of a tile: lanes of tensor memory
constexpr int LS_COLS = 256;         // most columns of the accumulator: units of BW rank rows of a pass
constexpr int LS_STAGES = 8;         // most stages
constexpr int LS_SMEM = 220 * 1024;  // most shared memory
constexpr int LS_TABLE = 128;        // stacks of at most so many adapters have their ranks and scales read ahead of the ids

struct alignas(16) ShrinkShared {
  uint64_t full[LS_STAGES], empty[LS_STAGES], done;
  uint32_t tmem_base;
  int abort_flag;
  alignas(16) int id[LS_ROWS];       // adapter of every row, read four at a time
  int at[LS_ROWS], steps[LS_ROWS];   // its first unit, and how many it has
  float scale[LS_ROWS];
  int step_table[LS_TABLE];
  float scale_table[LS_TABLE];
  int unit_row[LS_COLS / 16];        // first row of a unit in the stacked A
  int warp_units[4];
  int units;                         // of the whole tile
};

// A cluster multiplies the tile's rows with up to `most` units (BW rank rows of an adapter) as if they were the rows of one weight: D[row][unit, rank]. CTA c
// takes the c-th eighth of K's 64-wide blocks. A row keeps the columns of its own adapter: partial sums go to CTA row % 8, which adds them in
// ascending order. blockIdx.y: passes y, y + gridDim.y, ... over the tile's units.
template <int BW>
__global__ void __launch_bounds__(192)
lora_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const LoraArgs a, const float* __restrict__ scale, int scales,
                   __nv_bfloat16* __restrict__ t, int M, int K, int xrows, int most, int stages, int recv_off, int* status) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ ShrinkShared sh;
  constexpr int UNIT_BYTES = BW * 128;
  if (LS_SPLIT > 1) cluster_arrive_relaxed();            // "this CTA runs": waited on before the first store into a peer
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* recv = reinterpret_cast<float*>(ring + recv_off);          // partial sums: [unit][source CTA][16 rows][BW ranks]
  const int x_bytes = xrows * 128, stage_bytes = x_bytes + most * UNIT_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, crank = (int)cluster_ctarank();
  const int row0 = blockIdx.z * LS_ROWS, kblocks = (K + 63) / 64;
  const int kb0 = kblocks * crank / LS_SPLIT, kb1 = kblocks * (crank + 1) / LS_SPLIT;
  uint32_t tmem_cols = 32;
  while ((int)tmem_cols < BW * most) tmem_cols <<= 1;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmX); tma_prefetch_desc(&tmA);
    for (int i = 0; i < stages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
    mbar_init(&sh.done, 1);
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  const int e = threadIdx.x - 64;
  const bool table = a.adapters <= LS_TABLE;
  if (warp >= 2 && e < a.adapters && table) { sh.step_table[e] = lora_steps(a, e); sh.scale_table[e] = scales ? 0.f : scale[e]; }
  pdl_wait();
  // Tensor memory behind the wait, as in gemm_bf16.cu: what is taken here is not in the way of a kernel that still has to take its own. With it in hand the
  // kernel behind this one may start: it is told that X and the ids are done, takes its own and streams its weights meanwhile.
  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, tmem_cols); tmem_relinquish();
    if (lane == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) lora_set_ready(a);
    __syncwarp();
    pdl_trigger();
  }
  if (warp >= 2) {
    // distinct adapters of the tile and where their units lie in the tile's list, in the order of their first rows
    int id = row0 + e < M ? a.ids[row0 + e] : -1;
    if (id >= a.adapters) { if (blockIdx.y == 0 && crank == 0) set_status(status, KID_LORA, FF_ERR_BOUNDS, row0 + e, id); id = -1; }
    sh.id[e] = id;
    int steps = 0;
    float f = 0.f;
    if (!table && id >= 0) { steps = lora_steps(a, id); f = scales ? 0.f : scale[id]; }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (table && id >= 0) { steps = sh.step_table[id]; f = sh.scale_table[id]; }
    int first = e;
    if (id >= 0)
      for (int j = 0; j < first; j += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&sh.id[j]);
        if (v.w == id) first = min(first, j + 3);
        if (v.z == id) first = min(first, j + 2);
        if (v.y == id) first = min(first, j + 1);
        if (v.x == id) first = min(first, j);
      }
    const int own = first == e ? steps : 0;
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
    if (lane == 31) sh.warp_units[warp - 2] = upto;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    int before = upto - own, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) { if (w < warp - 2) before += sh.warp_units[w]; all += sh.warp_units[w]; }
    sh.at[e] = before;
    sh.steps[e] = steps;
    sh.scale[e] = f;
    if (e == 0) sh.units = all;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int shared_at = sh.at[first];
    asm volatile("bar.sync 1, 128;" ::: "memory");
    sh.at[e] = shared_at;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem_base;
  volatile int* abort_flag = &sh.abort_flag;
  const int units = sh.units;
  RingPos rp;
  uint32_t pass_it = 0;
  cluster_wait();
  for (int u0 = blockIdx.y * most; u0 < units; u0 += gridDim.y * most, ++pass_it) {
    const int n = min(most, units - u0);
    // the pass's units; every row of an adapter names the same ones
    if (warp >= 2) {
      const int at = sh.at[e], steps = sh.steps[e];
      for (int s = max(0, u0 - at); s < steps && at + s < u0 + n; ++s) sh.unit_row[at + s - u0] = sh.id[e] * a.R + BW * s;
    }
    __syncthreads();
    if (warp == 0) {
      if (elect_one()) {
        RingPos at = rp;
        for (int kb = kb0; kb < kb1; ++kb, at.next(stages)) {
          if (!mbar_wait(&sh.empty[at.s], at.ph ^ 1, abort_flag, status, KID_LORA, 1)) break;
          mbar_expect_tx(&sh.full[at.s], x_bytes + n * UNIT_BYTES);
          uint8_t* sa = ring + at.s * stage_bytes;
          tma_load_2d(sa, &tmX, &sh.full[at.s], kb * 64, row0);
          for (int j = 0; j < n; ++j) tma_load_2d(sa + x_bytes + j * UNIT_BYTES, &tmA, &sh.full[at.s], kb * 64, sh.unit_row[j]);
        }
      }
    } else if (warp == 1) {
      if (elect_one()) {
        const uint32_t idesc = umma_idesc(1, 1, 0, 0, LS_ROWS, BW * n);
        RingPos at = rp;
        for (int kb = kb0; kb < kb1; ++kb, at.next(stages)) {
          if (!mbar_wait(&sh.full[at.s], at.ph, abort_flag, status, KID_LORA, 2)) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(ring + at.s * stage_bytes);
          const uint64_t da = umma_desc_sw128(sa, 16, 1024), db = umma_desc_sw128(sa + x_bytes, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16(tmem_base, da + 2 * k, db + 2 * k, idesc, kb > kb0 || k > 0);
          umma_commit(&sh.empty[at.s]);
        }
        umma_commit(&sh.done);
      }
    }
    rp.skip(kb1 - kb0, stages);
    if (warp >= 2 && kb1 > kb0) {
      const bool ok = mbar_wait(&sh.done, pass_it & 1, abort_flag, status, KID_LORA, 3);
      tc_fence_after();
      __syncwarp();
      const int q = warp & 3, row = q * 32 + lane, at = sh.at[row] - u0, steps = sh.steps[row];
      for (int j = 0; j < n; ++j) {
        const bool mine = ok && j >= at && j < at + steps;
        if (!__any_sync(0xffffffffu, mine)) continue;
#pragma unroll
        for (int c = 0; c < BW; c += 16) {
          uint32_t r[16];
          tmem_ld_x16(tmem_base + (uint32_t(q * 32) << 16) + BW * j + c, r);
          tmem_ld_wait();
          if (mine) {
            const uint32_t dst = dsmem_addr(smem_u32(recv + ((j * LS_SPLIT + crank) * 16 + (row >> 3)) * BW + c), row & 7);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st_dsmem_f4(dst + 16 * i, make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3])));
          }
          __syncwarp();
        }
      }
      tc_fence_before();
    }
    __syncwarp();
    cluster_sync_all();
    // rows crank, crank + 8, ...: four ranks per thread
    constexpr int QUADS = BW / 4;
    for (int i = threadIdx.x; i < n * 16 * QUADS; i += 192) {
      const int j = i / (16 * QUADS), row = (i / QUADS % 16) * 8 + crank, quad = i % QUADS, step = u0 + j - sh.at[row];
      if (row0 + row >= M || step < 0 || step >= sh.steps[row]) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < LS_SPLIT; ++c) {
        if (kblocks * (c + 1) / LS_SPLIT == kblocks * c / LS_SPLIT) continue;          // a CTA without K blocks sent nothing
        const float4 x = *reinterpret_cast<const float4*>(recv + ((j * LS_SPLIT + c) * 16 + (row >> 3)) * BW + 4 * quad);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      }
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = scales ? scale[(size_t)sh.id[row] * a.R + BW * step + 4 * quad + k] : sh.scale[row];
      float low[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] *= f[k];
        const float h = __bfloat162float(__float2bfloat16(v[k]));
        low[k] = isinf(h) ? 0.f : v[k] - h;              // an infinite first word has no second: infinity less infinity would be NaN
      }
      __nv_bfloat16* dst = t + (size_t)(row0 + row) * 2 * a.R + BW * step + 4 * quad;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      *reinterpret_cast<uint2*>(dst + a.R) = make_uint2(pack_bf16x2(low[0], low[1]), pack_bf16x2(low[2], low[3]));
    }
    if (u0 + (int)gridDim.y * most < units) cluster_sync_all();      // the next pass's partial sums come to the same place
  }
  __syncthreads();
  if (sh.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) { __nanosleep(1000); }
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, tmem_cols); }
}

}  // namespace ff
using namespace ff;

// Everything of a call, written by the Python side (lora_ops._Lora has the same fields in the same order).
struct FfLora {
  const void *x, *w;
  void* y;
  const void *a, *b;
  const float* scale;
  const int *ranks, *ids, *part_of;
  void* t;                             // [M, 2R] BF16, and a word of 64 bits
  float* scratch;                      // scratch and counters of the decode product
  int *counters, *status;
  const float* cos_sin;
  const int* slots;
  void *kcache, *vcache;
  long long scratch_bytes, counter_bytes, call;          // call: a number that no other call has
  int M, N, K, ldx, ldw, ldy, R, adapters, parts, step, epi, gate, scales;  // step: ranks of a step of a fused projection; scales: 1 with a scale per rank row
  float limit;
  int hq, hkv, rot_dim, block_size, num_blocks;
};

static unsigned long long* lora_word(const FfLora& c) { return reinterpret_cast<unsigned long long*>(static_cast<__nv_bfloat16*>(c.t) + (size_t)c.M * 2 * c.R); }

static int lora_shrink(const FfLora& c, int bw, cudaStream_t stream) {
  const int tiles = (c.M + LS_ROWS - 1) / LS_ROWS, xrows = c.M < LS_ROWS ? (c.M + 15) / 16 * 16 : LS_ROWS, per = c.R / bw;
  const int rows = c.M < LS_ROWS ? c.M : LS_ROWS, units = (rows < c.adapters ? rows : c.adapters) * per;          // most that a tile can have
  // passes side by side: where tiles are few, so many that two CTAs stand on every SM
  const int lanes = 2 * sm_count() / (LS_SPLIT * tiles) > 1 ? 2 * sm_count() / (LS_SPLIT * tiles) : 1;
  int most = (units + lanes - 1) / lanes;
  // prompts have few adapters in a tile: passes as wide as one of them, and a ring of several stages
  if (c.M > LS_ROWS) most = per < 64 / bw ? 64 / bw : per > 128 / bw ? 128 / bw : per;
  most = most > units ? units : most;
  most = most > LS_COLS / bw ? LS_COLS / bw : most;
  // two stages and the partial sums have to fit an SM: 128 rows leave room for passes of 224 columns
  auto stage_of = [&](int n) { return xrows * 128 + n * bw * 128; };
  auto recv_of = [&](int n) { return n * LS_SPLIT * 16 * bw * 4; };
  while (most > 1 && 1024 + 2 * stage_of(most) + recv_of(most) > LS_SMEM) --most;
  int passes = (units + most - 1) / most;
  passes = passes < lanes ? passes : lanes;
  CUtensorMap tmX, tmA;
  if (int e = make_tmap_2d(&tmX, c.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c.K, c.M, (uint64_t)c.ldx * 2, 64, xrows)) return e;
  if (int e = make_tmap_2d(&tmA, c.a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c.K, (uint64_t)c.adapters * c.R, (uint64_t)c.K * 2, 64, bw)) return e;
  const int stage = stage_of(most), kb = ((c.K + 63) / 64 + LS_SPLIT - 1) / LS_SPLIT, recv = recv_of(most);
  // two CTAs on an SM for prompts; for decode rows so little that one fits beside a CTA of the product (7 rows, 4096 x 14336: 29.0 -> 24.6 us)
  int stages = ((c.M > LS_ROWS ? 108 : 40) * 1024 - recv) / stage;
  stages = stages > LS_STAGES ? LS_STAGES : stages < 2 ? 2 : stages;
  stages = stages > kb ? (kb < 2 ? 2 : kb) : stages;
  // the instruction reads 128 rows of X, past the loaded ones into what lies behind them
  const int slack = stage < LS_ROWS * 128 ? LS_ROWS * 128 - stage : 0, recv_off = stages * stage, smem = 1024 + recv_off + (recv > slack ? recv : slack);
  auto kern = bw == 32 ? lora_shrink_kernel<32> : lora_shrink_kernel<16>;
  if (int e = opt_in_smem(kern, LS_SMEM)) return e;
  const LoraArgs args = {c.ids, c.ranks, c.part_of, c.adapters, c.R, c.parts, bw, lora_word(c), (unsigned long long)c.call};
  return launch_pdl(kern, dim3(LS_SPLIT, passes, tiles), dim3(192), smem, stream, LS_SPLIT, tmX, tmA, args, c.scale, c.scales,
                    static_cast<__nv_bfloat16*>(c.t), c.M, c.K, xrows, most, stages, recv_off, c.status);
}

// Y = epi(X W^T + delta). epi 0: BF16 rows of N; 1: gate and up (interleaved per 64) with the activation `gate` / `limit`, rows of N / 2; 2: rotary embedding
// and cache write of a QKV product. FF_HOST_TOO_LARGE: scratch or counters are smaller than ff_gemm_skinny_plan(_epi) asks for; nothing was launched.
FF_EXPORT int ff_linear_lora(const FfLora* p, cudaStream_t stream) {
  if (p == nullptr) return FF_HOST_BAD_SHAPE;
  const FfLora& c = *p;
  if (c.M <= 0 || c.N <= 0 || c.K <= 0 || c.ldx < c.K || c.ldw < c.K || c.R <= 0 || c.R % 16 || c.R > 1024 || c.adapters <= 0) return FF_HOST_BAD_SHAPE;
  if (c.epi < 0 || c.epi > 2 || (c.part_of != nullptr && (c.parts <= 0 || (c.step != 16 && c.step != 32) || c.R % c.step))) return FF_HOST_BAD_SHAPE;
  if ((long long)c.adapters * c.N > 0x7fffffffll || (long long)c.adapters * c.R > 0x7fffffffll || (c.M + LS_ROWS - 1) / LS_ROWS > 65535) return FF_HOST_TOO_LARGE;
  if (c.epi == 1 && c.gate != 0 && c.gate != 3 && c.gate != 5) return FF_HOST_UNSUPPORTED;
  if (c.a == nullptr || c.b == nullptr || c.scale == nullptr || c.ids == nullptr || c.t == nullptr) return FF_HOST_BAD_SHAPE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.w) | reinterpret_cast<uintptr_t>(c.a) | reinterpret_cast<uintptr_t>(c.b) |
                        reinterpret_cast<uintptr_t>(c.t);
  if (all & 15 || c.K % 8 || c.ldx % 8 || c.ldw % 8) return FF_HOST_BAD_ALIGN;
  const QkvRope rope = {c.cos_sin, c.slots, c.kcache, c.vcache, c.hq, c.hkv, c.rot_dim, c.block_size, c.num_blocks};
  // units of 32 ranks are one copy where two of 16 are two; a stack of 16 has no more, and the steps of a fused projection are given
  const int bw = c.part_of != nullptr ? c.step : c.R % 32 ? 16 : 32;
  const LoraCall lora = {c.t, c.b, c.ids, c.ranks, c.part_of, c.adapters, c.R, c.parts, bw, lora_word(c), (unsigned long long)c.call};
  if (c.M > FF_SKINNY_MAX_ROWS) {
    if (c.N % 8 || c.ldy % 8 || (reinterpret_cast<uintptr_t>(c.y) & 15)) return FF_HOST_BAD_ALIGN;       // before anything is launched
    if (int e = lora_shrink(c, bw, stream)) return e;
    return ff_gemm_bf16_lora(c.x, c.w, c.y, c.M, c.N, c.K, c.ldx, c.ldw, c.ldy, &lora, c.epi == 2 ? 3 : c.epi, c.gate, c.limit, c.epi == 2 ? &rope : nullptr,
                             c.status, stream);
  }
  long long sb = 0, cb = 0;
  const int grid = c.epi ? ff_gemm_skinny_plan_epi(c.M, c.N, c.K, c.epi, &sb, &cb) : ff_gemm_skinny_plan(c.M, c.N, c.K, &sb, &cb);
  if (grid < 0) return grid;
  if (sb > c.scratch_bytes || cb > c.counter_bytes) return FF_HOST_TOO_LARGE;
  if (int e = lora_shrink(c, bw, stream)) return e;
  return ff_gemm_skinny_lora(c.x, c.w, c.y, c.M, c.N, c.K, c.ldx, c.ldw, c.ldy, grid, c.scratch, c.counters, &lora, c.epi, c.gate, c.limit,
                             c.epi == 2 ? &rope : nullptr, c.status, stream);
}
