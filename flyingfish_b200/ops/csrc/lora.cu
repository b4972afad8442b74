// Low-rank adapters of many requests beside a shared projection:  Y[M,N] = X W^T + delta,  delta_r = B_a (s_a A_a x_r)  for the
// adapter a = ids[r] of row r, no delta where ids[r] is negative. A stack holds the adapters of one projection: A [adapters, R, K],
// B [adapters, N, R], scales and ranks (rank rows behind an adapter's own are zero and not read). R is a multiple of 16.
//
//   lora_shrink_kernel   t_r = s_a A_a x_r          [M, 2R]: every value as two BF16 words, t = high + low
//   lora_expand_kernel   delta_r = B_a t_r          [M, ldd] FP32
//   gemm_skinny.cu       the product with W; its epilogue adds delta to the FP32 sums and rounds once
//
// A row is multiplied with its own adapter and nothing else: rows of a tile are listed by adapter first, and the tokens lie on the N side of
// mma.sync m16n8k16, so that a lone row costs 8 columns, a row without an adapter nothing, and what an adapter's weights hold (infinities
// included) reaches its own rows alone. Both kernels move bytes: A and B are read once per tile of rows and there are 16 to 256 of their
// rows or columns, so the arithmetic is no concern.
//
// t in two BF16 words: the second product's tensor instructions take BF16, one word would leave 2^-9 of t, two leave 2^-17 or less. B meets
// both words in one accumulator.
//
// The order of every sum depends on K and R alone, not on the batch or on where in it a row lies: a row's bits do not change with its neighbours.
#include "mma_sync.cuh"
#include "host_util.h"
#include "launchers.h"

namespace ff {

constexpr int LORA_C = 8;            // CTAs of a cluster share K
constexpr int LORA_WARPS = 8;

struct LoraStack {
  const __nv_bfloat16* a; const __nv_bfloat16* b; const float* scale; const int* ranks;
  int adapters, R;
};

__device__ __forceinline__ int lora_rank(const LoraStack& st, int adapter) {
  const int r = st.ranks == nullptr ? st.R : min(max(st.ranks[adapter], 0), st.R);
  return (r + 15) & ~15;
}

// The rows row0 .. row0 + 32 H of a tile by adapter: next() walks the distinct adapters in the order of their first rows. Warp-wide; lane i looks after
// rows row0 + i + 32 h.
template <int H>
struct RowGroups {
  int id[H];
  uint32_t left[H], mine[H];
  int adapter, count;
  __device__ __forceinline__ void load(const int* ids, int row0, int M, int adapters, int lane, int kid, int* status) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int r = row0 + 32 * h + lane;
      id[h] = r < M ? ids[r] : -1;
      if (id[h] >= adapters) { set_status(status, kid, FF_ERR_BOUNDS, r, id[h]); id[h] = -1; }
      left[h] = __ballot_sync(0xffffffffu, id[h] >= 0);
    }
  }
  __device__ __forceinline__ bool next() {
    adapter = -1;
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (adapter < 0 && left[h]) adapter = __shfl_sync(0xffffffffu, id[h], __ffs(left[h]) - 1);
    if (adapter < 0) return false;
    count = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      mine[h] = __ballot_sync(0xffffffffu, id[h] == adapter);
      left[h] &= ~mine[h];
      count += __popc(mine[h]);
    }
    return true;
  }
  // rows of the group in ascending order
  __device__ __forceinline__ void list(int* rows, int row0, int lane) const {
    int before = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (mine[h] >> lane & 1) rows[before + __popc(mine[h] & ((1u << lane) - 1))] = row0 + 32 * h + lane;
      before += __popc(mine[h]);
    }
  }
};

// A cluster multiplies RCH * 16 rank rows of an adapter with up to 8 NT of the tile's rows. CTA c and warp w take the 64-wide blocks of K number 8 c + w,
// + 64, ...; partial sums meet in shared memory, warps first, then CTAs, in ascending order. Operands go from global memory into the
// fragments: a lane loads 16 bytes of a row, elements 8 q .. 8 q + 7 of 32 along K, and both operands take them as the K indices of two
// instructions in the same (permuted) order.
template <int NT, int RCH>
__global__ void __launch_bounds__(32 * LORA_WARPS)
lora_shrink_kernel(const __nv_bfloat16* __restrict__ x, LoraStack st, const int* __restrict__ ids, __nv_bfloat16* __restrict__ t, int M, int K, int ldx,
                   int* status) {
  constexpr int H = NT / 4, P = 8 * NT + 8;           // pitch: 8-byte stores of 16 lanes fall into distinct banks
  __shared__ float red[LORA_WARPS][16][P];
  __shared__ float part[16 * RCH][P];
  __shared__ int lists[LORA_WARPS][8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int crank = (int)cluster_ctarank(), row0 = blockIdx.z * 8 * NT, chunks = (st.R + 16 * RCH - 1) / (16 * RCH);
  const int slot0 = blockIdx.y / chunks, slots = gridDim.y / chunks, rank0 = (blockIdx.y % chunks) * 16 * RCH;
  const int kblocks = (K + 63) / 64;
  int* list = lists[warp];
  pdl_wait();
  pdl_trigger();                                      // behind the wait: a kernel that starts now finds all of x
  RowGroups<H> rg;
  rg.load(ids, row0, M, st.adapters, lane, KID_LORA, status);
  for (int s = 0; rg.next(); ++s) {
    if (s % slots != slot0) continue;
    const int rank = lora_rank(st, rg.adapter), count = rg.count;
    if (rank0 >= rank) continue;
    __syncwarp();
    rg.list(list, row0, lane);
    __syncwarp();
    const int nt = (count + 7) >> 3;
    const __nv_bfloat16* arow[RCH][2];
#pragma unroll
    for (int c = 0; c < RCH; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = rank0 + 16 * c + 8 * h + g;
        arow[c][h] = r < st.R ? st.a + ((size_t)rg.adapter * st.R + r) * K : nullptr;
      }
    const __nv_bfloat16* xrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xrow[j] = 8 * j + g < count ? x + (size_t)list[8 * j + g] * ldx : nullptr;
    float acc[RCH][NT][4];
#pragma unroll
    for (int c = 0; c < RCH; ++c)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][j][e] = 0.f;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int kb = crank * LORA_WARPS + warp; kb < kblocks; kb += LORA_C * LORA_WARPS) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kb * 64 + h * 32 + q * 8;
        uint4 av[RCH][2], xv[NT];
#pragma unroll
        for (int c = 0; c < RCH; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) av[c][e] = k < K && arow[c][e] != nullptr ? __ldg(reinterpret_cast<const uint4*>(arow[c][e] + k)) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j) xv[j] = k < K && xrow[j] != nullptr ? __ldg(reinterpret_cast<const uint4*>(xrow[j] + k)) : zero;
#pragma unroll
        for (int c = 0; c < RCH; ++c) {
          const uint32_t a0[4] = {av[c][0].x, av[c][1].x, av[c][0].y, av[c][1].y}, a1[4] = {av[c][0].z, av[c][1].z, av[c][0].w, av[c][1].w};
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (j < nt) { ms_mma(acc[c][j], a0, xv[j].x, xv[j].y); ms_mma(acc[c][j], a1, xv[j].z, xv[j].w); }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < RCH; ++c) {
      if (c) __syncthreads();                         // the sums of the chunk before have been read
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (j < nt) {
          *reinterpret_cast<float2*>(&red[warp][g][8 * j + 2 * q]) = make_float2(acc[c][j][0], acc[c][j][1]);
          *reinterpret_cast<float2*>(&red[warp][8 + g][8 * j + 2 * q]) = make_float2(acc[c][j][2], acc[c][j][3]);
        }
      __syncthreads();
      for (int i = threadIdx.x; i < 16 * 8 * NT; i += 32 * LORA_WARPS) {
        const int r = i / (8 * NT), p = i % (8 * NT);
        if (p >= count) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < LORA_WARPS; ++w) v += red[w][r][p];
        part[16 * c + r][p] = v;
      }
    }
    cluster_sync_all();
    const float scale = st.scale[rg.adapter];
    for (int i = crank * 32 * LORA_WARPS + threadIdx.x; i < 16 * RCH * count; i += LORA_C * 32 * LORA_WARPS) {
      const int p = i / (16 * RCH), r = i % (16 * RCH);
      const uint32_t at = smem_u32(&part[r][p]);
      float in[LORA_C], v = 0.f;
#pragma unroll
      for (int c = 0; c < LORA_C; ++c) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(in[c]) : "r"(dsmem_addr(at, c)) : "memory");
#pragma unroll
      for (int c = 0; c < LORA_C; ++c) v += in[c];
      v *= scale;
      if (rank0 + r < st.R) {
        const __nv_bfloat16 high = __float2bfloat16(v);
        __nv_bfloat16* dst = t + (size_t)list[p] * 2 * st.R + rank0 + r;
        dst[0] = high;
        // an infinite first word has no second: infinity less infinity would be NaN
        dst[st.R] = __hisinf(high) ? __float2bfloat16(0.f) : __float2bfloat16(v - __bfloat162float(high));
      }
    }
    cluster_sync_all();                               // `part` is read by the peers until here
  }
}

// A warp multiplies 16 columns of B_a with up to 64 rows of a tile (8 columns of the instruction per 8 rows). part_of, where given: B of a fused
// projection is zero outside the 16-wide steps s = part_of[column / 64] (mod parts) of its R, and only those are read.
__global__ void __launch_bounds__(256)
lora_expand_kernel(const __nv_bfloat16* __restrict__ t, LoraStack st, const int* __restrict__ ids, const int* __restrict__ part_of, int parts,
                   float* __restrict__ delta, int M, int N, int ldd, int cols, int* status) {
  __shared__ int lists[8][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int row0 = blockIdx.z * 64, slots = gridDim.y;
  int* list = lists[warp];
  pdl_wait();
  pdl_trigger();
  RowGroups<2> rg;
  rg.load(ids, row0, M, st.adapters, lane, KID_LORA, status);
  for (int s = 0; rg.next(); ++s) {
    if (s % slots != (int)blockIdx.y) continue;
    const int steps = lora_rank(st, rg.adapter) / 16, count = rg.count, nt = (count + 7) >> 3;
    __syncwarp();
    rg.list(list, row0, lane);
    __syncwarp();
    const __nv_bfloat16* trow[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) trow[j] = 8 * j + g < count ? t + (size_t)list[8 * j + g] * 2 * st.R + 4 * q : nullptr;
    const uint2 zero = make_uint2(0, 0);
    for (int n0 = blockIdx.x * cols + 16 * warp; n0 < min(N, (int)(blockIdx.x + 1) * cols); n0 += 16 * 8) {
      const int first = part_of == nullptr ? 0 : part_of[n0 >> 6], by = part_of == nullptr ? 1 : parts;
      const __nv_bfloat16* b0 = n0 + g < N ? st.b + ((size_t)rg.adapter * N + n0 + g) * st.R + 4 * q : nullptr;
      const __nv_bfloat16* b1 = n0 + 8 + g < N ? st.b + ((size_t)rg.adapter * N + n0 + 8 + g) * st.R + 4 * q : nullptr;
      float acc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
      for (int k = first; k < steps; k += by) {
        const uint2 u = b0 != nullptr ? __ldg(reinterpret_cast<const uint2*>(b0 + 16 * k)) : zero;
        const uint2 v = b1 != nullptr ? __ldg(reinterpret_cast<const uint2*>(b1 + 16 * k)) : zero;
        const uint32_t a[4] = {u.x, v.x, u.y, v.y};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < nt) {
            const uint2 hi = trow[j] != nullptr ? *reinterpret_cast<const uint2*>(trow[j] + 16 * k) : zero;
            const uint2 lo = trow[j] != nullptr ? *reinterpret_cast<const uint2*>(trow[j] + 16 * k + st.R) : zero;
            ms_mma(acc[j], a, hi.x, hi.y);
            ms_mma(acc[j], a, lo.x, lo.y);
          }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int p = 8 * j + 2 * q + e;
          if (p < count) {
            float* dst = delta + (size_t)list[p] * ldd + n0 + g;
            if (n0 + g < N) dst[0] = acc[j][e];
            if (n0 + 8 + g < N) dst[8] = acc[j][2 + e];
          }
        }
    }
  }
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
  void* t;                             // [M, 2R] BF16
  float *delta, *scratch;              // delta: [delta_rows, ldd]; scratch and counters: those of the decode product
  int *counters, *status;
  const float* cos_sin;
  const int* slots;
  void *kcache, *vcache;
  long long scratch_bytes, counter_bytes;
  int M, N, K, ldx, ldw, ldy, ldd, delta_rows, R, adapters, parts, epi, gate;
  float limit;
  int hq, hkv, rot_dim, block_size, num_blocks;
};

static int lora_shrink(const FfLora& c, const __nv_bfloat16* x, const int* ids, __nv_bfloat16* t, int M, cudaStream_t stream) {
  const LoraStack st = {static_cast<const __nv_bfloat16*>(c.a), nullptr, c.scale, c.ranks, c.adapters, c.R};
  const bool few = M <= 128;
  const int rows = few ? 32 : 64, tiles = (M + rows - 1) / rows;
  int slots = few ? rows : 4;
  slots = slots < c.adapters ? slots : c.adapters;
  slots = slots < M ? slots : M;
  const int rch = c.R == 16 ? 1 : 2, chunks = (c.R + 16 * rch - 1) / (16 * rch);
  auto kern = few ? (rch == 1 ? lora_shrink_kernel<4, 1> : lora_shrink_kernel<4, 2>) : (rch == 1 ? lora_shrink_kernel<8, 1> : lora_shrink_kernel<8, 2>);
  return launch_pdl(kern, dim3(LORA_C, slots * chunks, tiles), dim3(32 * LORA_WARPS), 0, stream, LORA_C, x, st, ids, t, M, c.K, c.ldx, c.status);
}

static int lora_expand(const FfLora& c, const __nv_bfloat16* t, const int* ids, int M, cudaStream_t stream) {
  const LoraStack st = {nullptr, static_cast<const __nv_bfloat16*>(c.b), nullptr, c.ranks, c.adapters, c.R};
  const int tiles = (M + 63) / 64, cols = M <= 128 ? 128 : 1024, groups = (c.N + cols - 1) / cols;
  int slots = (sm_count() * 8 + groups * tiles - 1) / (groups * tiles);
  slots = slots < 64 ? slots : 64;
  slots = slots < c.adapters ? slots : c.adapters;
  slots = slots < M ? slots : M;
  return launch_pdl(lora_expand_kernel, dim3(groups, slots, tiles), dim3(256), 0, stream, 1, t, st, ids, c.part_of, c.parts, c.delta, M, c.N, c.ldd, cols,
                    c.status);
}

// Y = epi(X W^T + delta). epi 0: BF16 rows of N; 1: gate and up (interleaved per 64) with the activation `gate` / `limit`, rows of N / 2; 2: rotary embedding
// and cache write of a QKV product. Rows are done delta_rows at a time (all at once up to 128). FF_HOST_TOO_LARGE: scratch or counters are
// smaller than ff_gemm_skinny_plan(_epi) asks for; nothing was launched.
FF_EXPORT int ff_linear_lora(const FfLora* p, cudaStream_t stream) {
  if (p == nullptr) return FF_HOST_BAD_SHAPE;
  const FfLora& c = *p;
  if (c.M <= 0 || c.N <= 0 || c.K <= 0 || c.ldx < c.K || c.ldw < c.K || c.R <= 0 || c.R % 16 || c.R > 1024 || c.adapters <= 0 || c.delta_rows <= 0) return FF_HOST_BAD_SHAPE;
  if (c.epi < 0 || c.epi > 2 || (c.part_of != nullptr && c.parts <= 0) || c.ldd < (c.N + 7) / 8 * 8) return FF_HOST_BAD_SHAPE;
  if (c.epi == 1 && c.gate != 0 && c.gate != 3 && c.gate != 5) return FF_HOST_UNSUPPORTED;
  if (c.a == nullptr || c.b == nullptr || c.scale == nullptr || c.ids == nullptr || c.t == nullptr || c.delta == nullptr) return FF_HOST_BAD_SHAPE;
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.w) | reinterpret_cast<uintptr_t>(c.a) | reinterpret_cast<uintptr_t>(c.b) |
                        reinterpret_cast<uintptr_t>(c.t) | reinterpret_cast<uintptr_t>(c.delta);
  if (all & 15 || c.K % 8 || c.ldx % 8 || c.ldw % 8 || c.ldd % 8) return FF_HOST_BAD_ALIGN;
  const QkvRope rope = {c.cos_sin, c.slots, c.kcache, c.vcache, c.hq, c.hkv, c.rot_dim, c.block_size, c.num_blocks};
  __nv_bfloat16* t = static_cast<__nv_bfloat16*>(c.t);
  if (c.M <= FF_SKINNY_MAX_ROWS) {
    if (c.delta_rows < c.M) return FF_HOST_BAD_SHAPE;
    long long sb = 0, cb = 0;
    const int grid = c.epi ? ff_gemm_skinny_plan_epi(c.M, c.N, c.K, c.epi, &sb, &cb) : ff_gemm_skinny_plan(c.M, c.N, c.K, &sb, &cb);
    if (grid < 0) return grid;
    if (sb > c.scratch_bytes || cb > c.counter_bytes) return FF_HOST_TOO_LARGE;
    if (int e = lora_shrink(c, static_cast<const __nv_bfloat16*>(c.x), c.ids, t, c.M, stream)) return e;
    if (int e = lora_expand(c, t, c.ids, c.M, stream)) return e;
    return ff_gemm_skinny_delta(c.x, c.w, c.y, c.M, c.N, c.K, c.ldx, c.ldw, c.ldy, grid, c.scratch, c.counters, c.delta, c.ids, c.ldd, c.adapters, c.epi,
                                c.gate, c.limit, c.epi == 2 ? &rope : nullptr, c.status, stream);
  }
  for (int r0 = 0; r0 < c.M; r0 += c.delta_rows) {
    const int rows = c.M - r0 < c.delta_rows ? c.M - r0 : c.delta_rows;
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(c.x) + (size_t)r0 * c.ldx;
    QkvRope at = rope;
    if (c.epi == 2) { at.cos_sin += (size_t)r0 * c.rot_dim; at.slots += r0; }
    if (int e = lora_shrink(c, x, c.ids + r0, t, rows, stream)) return e;
    if (int e = lora_expand(c, t, c.ids + r0, rows, stream)) return e;
    if (int e = ff_gemm_bf16_delta(x, c.w, static_cast<__nv_bfloat16*>(c.y) + (size_t)r0 * c.ldy, rows, c.N, c.K, c.ldx, c.ldw, c.ldy, c.delta, c.ids + r0, c.ldd,
                                   c.adapters, c.epi == 2 ? 3 : c.epi, c.gate, c.limit, c.epi == 2 ? &at : nullptr, c.status, stream)) return e;
  }
  return FF_HOST_OK;
}
