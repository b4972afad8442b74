// Pages of a key / value cache that is held in 4 bits. A page is 64 tokens of one head of D = 64 or 128 elements; groups of 32
// neighbouring elements of a token share two BF16 numbers (scale, lo), an element stands for code * scale + lo:
//   lo = the group's least element, scale = RN_bf16((greatest - lo) / 15), code = RN_even((x - lo) / scale) in 0 .. 15
// (real numbers, one rounding each; scale and codes are 0 where the scale would be below the least normal BF16 number).
// 5 bits an element, 160 bytes a token and head of 128 for keys and values together where BF16 has 512.
//
// Layout of a page: 64 rows of D / 2 bytes of codes, then [64 tokens][D / 32] pairs (scale, lo). Element d = 32 j + 8 u + e:
//   keys    nibble e / 2 + 4 (e & 1) of 32-bit word u D / 32 + j of the token's row. Lane (g, t) of a warp reads words t D / 32 .. of the rows of two
//           tokens as its A fragments of mma.sync m16n8k16 (tokens x elements); masking a word at nibble i and i + 4 gives elements
//           8 t + 2 i and 8 t + 2 i + 1 of a group, in that order, as the queries are in memory.
//   values  nibble e / 2 of 16-bit unit j of chunk 2 u + (e & 1) (D / 16 bytes). Lane (g, t) reads chunk g of tokens 4 t .. 4 t + 3 as its fragments of
//           (elements x tokens). Rows and chunks are moved so that no two lanes of such a read meet a bank: token k lies at row
//           k ^ (k >> 3 & 1) with chunk c at c ^ 4 (k >> 2 & 1) for D = 128, at row k ^ (k >> 2 & 3) for D = 64.
#pragma once
#include "ptx.cuh"

namespace ff {

constexpr int KV4_PAGE = 64;
__host__ __device__ constexpr int kv4_code_bytes(int dim) { return KV4_PAGE * dim / 2; }
__host__ __device__ constexpr int kv4_page_bytes(int dim) { return KV4_PAGE * (dim / 2 + dim / 8); }

// Attention divides a page's (scale, lo) by a power of two of their size, so that FP16 holds them: the exponent field (2^-110) that it has at least, and how
// far below the greatest so far it may fall where sums are held over it.
constexpr int KV4_LEAST = 17, KV4_SPAN = 60;

// byte of 16-bit unit j of chunk c of token k's values
template <int D>
__device__ __forceinline__ int kv4_value_at(int k, int c, int j) {
  const int row = D == 128 ? k ^ ((k >> 3) & 1) : k ^ ((k >> 2) & 3);
  if (D == 128) c ^= ((k >> 2) & 1) << 2;
  return row * (D / 2) + c * (D / 16) + 2 * j;
}

__device__ __forceinline__ void kv4_sts(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void kv4_lds(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void kv4_lds(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t kv4_prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
__device__ __forceinline__ uint32_t kv4_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float kv4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void kv4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// by halves
__device__ __forceinline__ uint32_t kv4_mul2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
// the one of greater magnitude, with either's sign
__device__ __forceinline__ uint32_t kv4_maxabs2(uint32_t a, uint32_t b) { uint32_t r; asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
// over the warp
__device__ __forceinline__ uint32_t kv4_warp_max(uint32_t a) { return __reduce_max_sync(0xffffffffu, a); }

}  // namespace ff
