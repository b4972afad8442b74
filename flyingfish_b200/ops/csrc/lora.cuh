// What the products of gemm_skinny.cu and gemm_bf16.cu take to add low-rank adapters (lora.cu): the distinct adapters of a tile's rows as units of
// 16 ranks, the tensor maps of t and B, and tensor instructions that leave out lanes.
//
// A unit (adapter a, step s) is t[:, 16 s .. 16 s + 15] B_a[:, 16 s .. 16 s + 15]^T, accumulated behind the product's own K blocks into the same
// FP32 sums, for the rows of the adapter only: a row of the tile is a lane of tensor memory, and the instruction's mask of lanes leaves the others' sums
// alone, whatever t and B hold. So a tile takes any mix of adapters, a row without one gets the bits of the product alone, and what an adapter
// holds (infinities included) reaches its own rows only. t is two BF16 words per value (high, low), so a unit is two instructions. Two units
// share a stage of the ring: [high 0 | low 0 | high 1 | low 1] of t in the place of X, [B 0 | B 1] in the place of W, 32-byte swizzle.
#pragma once
#include "ptx.cuh"
#include "host_util.h"

namespace ff {

struct LoraArgs {
  const int *ids, *ranks, *part_of;    // ranks, part_of: may be null
  int adapters, R, parts;
};

struct LoraDev {                       // kernel parameter
  CUtensorMap t, b, b2;                // t [M, 2R]; B of all adapters [adapters * N, R], boxes of a tile's rows (b2: of the narrow tiles of a pair launch)
  LoraArgs a;
};
struct NoLora {};

__device__ __forceinline__ int lora_steps(const LoraArgs& a, int adapter) {
  const int r = a.ranks == nullptr ? a.R : min(max(a.ranks[adapter], 0), a.R);
  return (r + 15) >> 4;
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
// projection and see every parts-th step only. Of the `shares` CTAs that divide a tile's K, number `share` takes the units whose adapter + step leaves
// that remainder: where a row's units go depends on nothing but its adapter.
template <int H>
struct UnitWalk {
  RowGroups<H> rg;
  uint32_t mine[H];
  int adapter, step = 0, steps = 0, first, by, share, shares;
  __device__ __forceinline__ UnitWalk(const RowGroups<H>& all, int part, int parts, int share_, int shares_)
      : rg(all), first(part < 0 ? 0 : part), by(part < 0 ? 1 : parts), share(share_), shares(shares_) {}
  __device__ __forceinline__ bool next() {
    while (true) {
      for (; step < steps; step += by)
        if (shares == 1 || (unsigned)(adapter + step) % (unsigned)shares == (unsigned)share) return true;
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

// One or two units of a stage.
template <int H>
struct UnitPair {
  int n, adapter0, step0, adapter1, step1;
  uint32_t mine0[H], mine1[H];
  __device__ __forceinline__ bool next(UnitWalk<H>& w) {
    n = 0;
    if (!w.next()) return false;
    adapter0 = w.adapter; step0 = w.step; w.step += w.by; n = 1;
#pragma unroll
    for (int h = 0; h < H; ++h) mine0[h] = w.mine[h];
    if (w.next()) {
      adapter1 = w.adapter; step1 = w.step; w.step += w.by; n = 2;
#pragma unroll
      for (int h = 0; h < H; ++h) mine1[h] = w.mine[h];
    }
    return true;
  }
};

// the part that all of the columns [col0, col0 + width) lie in, or -1
__device__ __forceinline__ int lora_part(const LoraArgs& a, int col0, int width, int N) {
  if (a.part_of == nullptr) return -1;
  const int last = (min(col0 + width, N) - 1) >> 6;
  const int p = a.part_of[col0 >> 6];
  for (int i = (col0 >> 6) + 1; i <= last; ++i) if (a.part_of[i] != p) return -1;
  return p;
}

// K-major operand of 16 BF16 per row, 32-byte swizzle: rows of 32 bytes, groups of eight 256 bytes apart
__device__ __forceinline__ uint64_t umma_desc_sw32(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(256 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)6 << 61;      // SWIZZLE_32B
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

// tensor maps of t [M, 2R] (boxes of t_rows rows) and of B [adapters * N, R] (boxes of b_rows and b2_rows rows), 16 columns wide
inline int lora_maps(LoraDev& d, const void* t, const void* b, int M, int N, int t_rows, int b_rows, int b2_rows) {
  const uint64_t r = d.a.R;
  if (int e = make_tmap_2d(&d.t, t, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 2 * r, M, 4 * r, 16, t_rows, CU_TENSOR_MAP_SWIZZLE_32B)) return e;
  if (int e = make_tmap_2d(&d.b, b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, r, (uint64_t)d.a.adapters * N, 2 * r, 16, b_rows, CU_TENSOR_MAP_SWIZZLE_32B)) return e;
  return make_tmap_2d(&d.b2, b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, r, (uint64_t)d.a.adapters * N, 2 * r, 16, b2_rows, CU_TENSOR_MAP_SWIZZLE_32B);
}

}  // namespace ff
