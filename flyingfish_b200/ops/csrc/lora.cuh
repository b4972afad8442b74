// What the products of gemm_skinny.cu and gemm_bf16.cu take to add low-rank adapters (lora.cu): the distinct adapters of a tile's rows as units of
// BW = 16 or 32 ranks, the tensor maps of t and B, and tensor instructions that leave out lanes.
//
// A unit (adapter a, step s) is t[:, BW s ..] B_a[:, BW s ..]^T, BW columns of both, accumulated behind the product's own K blocks into the same FP32
// sums, for the rows of the adapter only: a row of the tile is a lane of tensor memory, and the instruction's mask of lanes leaves the others' sums
// alone, whatever t and B hold. So a tile takes any mix of adapters, a row without one gets the bits of the product alone, and what an adapter
// holds (infinities included) reaches its own rows only. t is two BF16 words per value (high, low), so 16 ranks are two instructions. Operands of BW
// columns lie in shared memory with a swizzle of their width.
#pragma once
#include "ptx.cuh"
#include "host_util.h"

namespace ff {

struct LoraArgs {
  const int *ids, *ranks, *part_of;    // ranks, part_of: may be null
  int adapters, R, parts, bw;
  unsigned long long *ready, call;     // where the call's number says that X and the ids are there
};

struct LoraDev {                       // kernel parameter
  CUtensorMap t, b, b2;                // t [M, 2R]; B of all adapters [adapters * N, R], boxes of a tile's rows (b2: of the narrow tiles of a pair launch)
  LoraArgs a;
};
struct NoLora {};

// What lies in front of a call -- X, the ids, tables of angles -- may reach the product before t does: the shrink waits for it, writes the call's number to
// `ready`, and only then lets the product start. A product that finds the number there has what it stands for (release and acquire, on the GPU) and puts its
// wait for the shrink in front of the first t; one that does not waits at once. Nobody polls. The word lies behind t and holds anything before a call: numbers
// are 63 bits, of a process's own, and the product's first CTA takes its call's away again, so that a replay does not find the number of the one before.
__device__ __forceinline__ void lora_set_ready(const LoraArgs& a) { asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(a.ready), "l"(a.call) : "memory"); }
__device__ __forceinline__ void lora_see_ready(const LoraArgs& a) {
  unsigned long long v;
  asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(a.ready) : "memory");
  if (v != a.call) pdl_wait();
}
// in front of loads by the TMA engine of what lora_see_ready() stands for
__device__ __forceinline__ void lora_ready_for_tma() { asm volatile("fence.proxy.async.global;" ::: "memory"); }
// one thread, behind a wait of its own; a CTA that looks later waits
__device__ __forceinline__ void lora_clear_ready(const LoraArgs& a) { if (blockIdx.x == 0) *a.ready = 0; }

__device__ __forceinline__ int lora_steps(const LoraArgs& a, int adapter) {
  const int r = a.ranks == nullptr ? a.R : min(max(a.ranks[adapter], 0), a.R);
  return (r + a.bw - 1) >> (a.bw == 32 ? 5 : 4);
}

// The rows row0 .. row0 + 32 H of a tile by adapter. Warp-wide; lane i looks after rows row0 + i + 32 h.
template <int H>
struct RowGroups {
  int id[H], steps[H];
  uint32_t left[H];
  __device__ __forceinline__ void load(const LoraArgs& a, int row0, int M, int lane, int* status) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int r = row0 + 32 * h + lane;
      id[h] = r < M ? a.ids[r] : -1;
      if (id[h] >= a.adapters) { set_status(status, KID_LORA, FF_ERR_BOUNDS, r, id[h]); id[h] = -1; }
    }
    load_steps(a);
    vote();
  }
  // load() in three parts, for a tile whose rows are looked up under the tile before
  __device__ __forceinline__ void load_ids(const LoraArgs& a, int row0, int M, int lane) {
#pragma unroll
    for (int h = 0; h < H; ++h) { const int r = row0 + 32 * h + lane; id[h] = r < M ? a.ids[r] : -1; }
  }
  __device__ __forceinline__ void load_steps(const LoraArgs& a) {
#pragma unroll
    for (int h = 0; h < H; ++h) steps[h] = (unsigned)id[h] < (unsigned)a.adapters ? lora_steps(a, id[h]) : 0;
  }
  __device__ __forceinline__ void vote() {
#pragma unroll
    for (int h = 0; h < H; ++h) left[h] = __ballot_sync(0xffffffffu, steps[h] > 0);
  }
};

// Units of a tile in turn: adapters in the order of their first rows, their steps ascending. part >= 0: the tile's columns lie in that part of a fused
// projection and see every parts-th step only.
template <int H>
struct UnitWalk {
  RowGroups<H> rg;
  uint32_t mine[H];
  int adapter, step = 0, steps = 0, first, by;
  __device__ __forceinline__ UnitWalk(const RowGroups<H>& all, int part, int parts) : rg(all), first(part < 0 ? 0 : part), by(part < 0 ? 1 : parts) {}
  __device__ __forceinline__ bool next() {
    while (true) {
      if (step < steps) return true;
      adapter = -1;
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (adapter < 0 && rg.left[h]) {
          const int lane = __ffs(rg.left[h]) - 1;
          adapter = __shfl_sync(0xffffffffu, rg.id[h], lane);
          steps = __shfl_sync(0xffffffffu, rg.steps[h], lane);
        }
      if (adapter < 0) return false;
#pragma unroll
      for (int h = 0; h < H; ++h) { mine[h] = __ballot_sync(0xffffffffu, rg.id[h] == adapter); rg.left[h] &= ~mine[h]; }
      step = first;
    }
  }
};

// The units of a stage: [high 0 | low 0 | high 1 | low 1] of t in the place of X, [B 0 | B 1] in the place of W, one unit of 32 ranks or up to two of 16.
template <int H>
struct UnitPair {
  int n, adapter0, step0, adapter1, step1;
  uint32_t mine0[H], mine1[H];
  __device__ __forceinline__ bool next(UnitWalk<H>& w, bool two) {
    n = 0;
    if (!w.next()) return false;
    adapter0 = w.adapter; step0 = w.step; w.step += w.by; n = 1;
#pragma unroll
    for (int h = 0; h < H; ++h) mine0[h] = w.mine[h];
    if (two && w.next()) {
      adapter1 = w.adapter; step1 = w.step; w.step += w.by; n = 2;
#pragma unroll
      for (int h = 0; h < H; ++h) mine1[h] = w.mine[h];
    }
    return true;
  }
};

// Decode products: one tile of up to 128 rows, whose adapters are listed once per CTA in shared memory by the epilogue's 128 threads while the weights stream.
// Units go step by step, so that t of a step is loaded once for all adapters (once for all tiles where there are no more steps than buffers); up to 64 / BW of
// a step's units share a stage of the ring. The threads that load and multiply walk lists of bits: one thread alone takes hundreds of cycles
// to find a unit among the adapters (64 rows with 64 adapters of rank 16, 6144 x 4096: 56 us with the search, 33.5 with the bits).
//
// Where a tile's K is divided among CTAs, a hash of the adapter and the step say whose a unit is: where a row's units go, and with it the order of its
// sums, depends on nothing but its adapter.
constexpr int LORA_LIST = 128, LORA_STEPS = 64;
struct LoraShare { int share, shares; };
struct LoraList {
  alignas(16) int id[LORA_LIST];
  alignas(16) uint32_t mine[LORA_LIST][4];             // rows of the n-th adapter
  alignas(16) uint32_t hits[3][LORA_STEPS][4];         // adapters with a unit of this step: of the whole tile, of this CTA's first and last share of a tile
  int row[LORA_LIST];                                  // first row of the n-th adapter in the stacked B
  int hash[LORA_LIST], most[LORA_LIST], index[LORA_LIST], warp_count[4], warp_steps[4];
  int count, steps;                                    // adapters, most steps of one
  alignas(8) uint64_t listed, t_full[2], t_empty[2];
};

// 128 threads, e = 0 .. 127; `listed` (4 arrivals) says that it is done.
__device__ __forceinline__ void lora_list(LoraList& l, const LoraArgs& a, int M, int N, int e, LoraShare first_share, LoraShare last_share, int* status) {
  const int warp = e >> 5, lane = e & 31;
  int id = e < M ? a.ids[e] : -1;
  if (id >= a.adapters) { if (blockIdx.x == 0) set_status(status, KID_LORA, FF_ERR_BOUNDS, e, id); id = -1; }
  const int steps = id >= 0 ? lora_steps(a, id) : 0;
  if (steps == 0) id = -1;
  l.id[e] = id;
  *reinterpret_cast<uint4*>(l.mine[e]) = make_uint4(0, 0, 0, 0);
  asm volatile("bar.sync 1, 128;" ::: "memory");
  int first = e;
  if (id >= 0)
    for (int j = 0; j < first; j += 4) {
      const int4 v = *reinterpret_cast<const int4*>(&l.id[j]);
      if (v.w == id) first = min(first, j + 3);
      if (v.z == id) first = min(first, j + 2);
      if (v.y == id) first = min(first, j + 1);
      if (v.x == id) first = min(first, j);
    }
  const bool leads = id >= 0 && first == e;
  const uint32_t vote = __ballot_sync(0xffffffffu, leads);
  const int most = (int)__reduce_max_sync(0xffffffffu, (unsigned)steps);
  if (lane == 0) { l.warp_count[warp] = __popc(vote); l.warp_steps[warp] = most; }
  asm volatile("bar.sync 1, 128;" ::: "memory");
  int at = __popc(vote & ((1u << lane) - 1));
  for (int w = 0; w < warp; ++w) at += l.warp_count[w];
  const int count = l.warp_count[0] + l.warp_count[1] + l.warp_count[2] + l.warp_count[3];
  const int all_steps = max(max(l.warp_steps[0], l.warp_steps[1]), max(l.warp_steps[2], l.warp_steps[3]));
  if (leads) { l.row[at] = id * N; l.hash[at] = (int)(((unsigned)id * 40503u) & 0xffffu); l.most[at] = steps; l.index[e] = at; }
  if (e == 0) { l.count = count; l.steps = all_steps; }
  asm volatile("bar.sync 1, 128;" ::: "memory");
  const uint32_t same = __match_any_sync(0xffffffffu, id);
  if (id >= 0 && lane == __ffs(same) - 1) l.mine[l.index[first]][warp] = same;
  // thread e: the e-th adapter
  const int mine = e < count ? l.most[e] : 0, hash = e < count ? l.hash[e] : 0;
  int r0 = hash * first_share.shares >> 16, r1 = hash * last_share.shares >> 16;
  for (int s = 0; s < all_steps; ++s) {
    const uint32_t whole = __ballot_sync(0xffffffffu, s < mine);
    const uint32_t one = __ballot_sync(0xffffffffu, s < mine && r0 == first_share.share), two = __ballot_sync(0xffffffffu, s < mine && r1 == last_share.share);
    if (lane == 0) { l.hits[0][s][warp] = whole; l.hits[1][s][warp] = one; l.hits[2][s][warp] = two; }
    if (++r0 == first_share.shares) r0 = 0;
    if (++r1 == last_share.shares) r1 = 0;
  }
  __syncwarp();
  if (lane == 0) mbar_arrive(&l.listed);
}

// the part that all of the columns [col0, col0 + width) lie in, or -1
__device__ __forceinline__ int lora_part(const LoraArgs& a, int col0, int width, int N) {
  if (a.part_of == nullptr) return -1;
  const int last = (min(col0 + width, N) - 1) >> 6;
  const int p = a.part_of[col0 >> 6];
  for (int i = (col0 >> 6) + 1; i <= last; ++i) if (a.part_of[i] != p) return -1;
  return p;
}

// K-major operand of BW BF16 per row, swizzle of the row's width: groups of eight rows 16 BW bytes apart
template <int BW>
__device__ __forceinline__ uint64_t umma_desc_narrow(uint32_t smem_addr) {
  static_assert(BW == 16 || BW == 32);
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)BW << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(BW == 16 ? 6 : 4) << 61;      // SWIZZLE_32B, SWIZZLE_64B
  return d;
}

// D[lanes] += A B, for the lanes (rows) of `mine`
__device__ __forceinline__ void umma_f16_lanes(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, const uint32_t (&mine)[4]) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7}, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(~mine[0]), "r"(~mine[1]), "r"(~mine[2]), "r"(~mine[3]) : "memory");
}
__device__ __forceinline__ void umma_f16_pair_lanes(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, const uint32_t (&mine)[8]) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(~mine[0]), "r"(~mine[1]), "r"(~mine[2]), "r"(~mine[3]), "r"(~mine[4]), "r"(~mine[5]),
      "r"(~mine[6]), "r"(~mine[7]) : "memory");
}

// a unit: both words of t (t_high, t_low) times B, in shared memory, for the lanes of `mine`
template <int BW>
__device__ __forceinline__ void umma_unit(uint32_t d_tmem, uint32_t t_high, uint32_t t_low, uint32_t b, uint32_t idesc, const uint32_t (&mine)[4]) {
  const uint64_t h = umma_desc_narrow<BW>(t_high), l = umma_desc_narrow<BW>(t_low), w = umma_desc_narrow<BW>(b);
#pragma unroll
  for (int k = 0; k < BW / 16; ++k) umma_f16_lanes(d_tmem, h + 2 * k, w + 2 * k, idesc, mine);
#pragma unroll
  for (int k = 0; k < BW / 16; ++k) umma_f16_lanes(d_tmem, l + 2 * k, w + 2 * k, idesc, mine);
}
template <int BW>
__device__ __forceinline__ void umma_unit_pair(uint32_t d_tmem, uint32_t t_high, uint32_t t_low, uint32_t b, uint32_t idesc, const uint32_t (&mine)[8]) {
  const uint64_t h = umma_desc_narrow<BW>(t_high), l = umma_desc_narrow<BW>(t_low), w = umma_desc_narrow<BW>(b);
#pragma unroll
  for (int k = 0; k < BW / 16; ++k) umma_f16_pair_lanes(d_tmem, h + 2 * k, w + 2 * k, idesc, mine);
#pragma unroll
  for (int k = 0; k < BW / 16; ++k) umma_f16_pair_lanes(d_tmem, l + 2 * k, w + 2 * k, idesc, mine);
}

// tensor maps of t [M, 2R] (boxes of t_rows rows) and of B [adapters * N, R] (boxes of b_rows and b2_rows rows), bw columns wide
inline int lora_maps(LoraDev& d, const void* t, const void* b, int M, int N, int t_rows, int b_rows, int b2_rows) {
  const uint64_t r = d.a.R;
  const CUtensorMapSwizzle sw = d.a.bw == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  if (int e = make_tmap_2d(&d.t, t, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 2 * r, M, 4 * r, d.a.bw, t_rows, sw)) return e;
  if (int e = make_tmap_2d(&d.b, b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, r, (uint64_t)d.a.adapters * N, 2 * r, d.a.bw, b_rows, sw)) return e;
  if (b2_rows == b_rows) { d.b2 = d.b; return FF_HOST_OK; }
  return make_tmap_2d(&d.b2, b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, r, (uint64_t)d.a.adapters * N, 2 * r, d.a.bw, b2_rows, sw);
}

}  // namespace ff
