// Attention over the 4-bit key / value cache (layout and format: kv4.cuh).
#include "kv4.cuh"
#include "host_util.h"
#include "mma_sync.cuh"

namespace ff {

constexpr float KV4_NONE = -3.0e38f;       // running maximum of a row that has seen no key

// the 8 x 8 matrix of 16-bit elements that the warp's registers hold by rows, transposed
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void kv4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float kv4_low(uint32_t w) { return __uint_as_float(w << 16); }              // BF16 in the lower / upper half
__device__ __forceinline__ float kv4_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float kv4_peer(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(dsmem_addr(smem_u32(p), (uint32_t)rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 kv4_peer2(const float* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(dsmem_addr(smem_u32(p), (uint32_t)rank)) : "memory");
  return v;
}
template <int NG>
__device__ __forceinline__ void kv4_words(uint32_t (&dst)[NG], uint32_t src) {
  if constexpr (NG == 4) kv4_lds(src, dst[0], dst[1], dst[2], dst[3]);
  else kv4_lds(src, dst[0], dst[1]);
}

// Rows of queries, a few per sequence (one in a decode step): the rows of one sequence times the query heads of one kv head are the columns of
//   S^T [keys x columns] = K Q^T        O^T [elements x columns] = V^T P^T
// so that the cache is the 16-row operand of mma.sync m16n8k16 and 8 columns are enough to fill an instruction. Codes go into the products as they are,
//   S = sum_j scale_j (q_j . n_j) + lo_j sum(q_j)          O_j = sum_k (p_k scale_kj) n_kj + sum_k p_k lo_kj
// for groups j of 32 elements. A code at bits 0 .. 3 of a 16-bit half is the FP16 number n 2^-24, at bits 4 .. 7 n 2^-20 (both subnormal, so exact and linear):
// four pairs of codes are four masks and one shift, and nothing has to be subtracted. The powers of two go into the queries (every other pair of elements, and
// a power per column that brings its greatest element to 2^14) and out of the results. Sums, maxima, the keys' scale and lo are FP32,
// and sum(q_j) is three BF16 parts of a product of its own, whose A operand is lo as it is. The sums of p lo are a product too.
// Rounded to FP16 are p, p scale and lo, 11 bits each, whatever size the values are: a warp divides scale and lo by a power of two that the greatest of the page
// lies at most KV4_KEPT binades below (and never above), its O is held over the same power and follows where that moves. Multiplied by 2^7, as p is, they fill
// FP16's range: p scale has 11 bits down to 2^-28 of what it can be, p and lo down to 2^-21; what is smaller is off by 2^-39 or 2^-32 of the page's
// greatest. BF16 would need no power, but has 8 bits of p scale, and code times scale is some three times a value. Values as they are, without the power: those of 2^-20 off by 8 %
// and more, a long tail of small weights behind a single great one by 1 to 10 % for values of 2^-10.
// A CTA has NT x 8 columns and a range of pages; every warp takes pages of its own, fetched by bulk copies into its two slots (keys, values),
// with its own running maximum, sum and O. The warps' results meet in shared memory, those of up to eight CTAs (splits) in that of
// their cluster, those of more in kv4_merge_kernel.
// Bound by issue slots, not by the 5 bits an element of traffic: three sequences of up to 131071 tokens, 64 / 8 heads: 102 us for 474 MB (4.6 TB/s of the 6.5 a copy
// reaches), 1267 instructions a page and warp, 72 of them for the power of two (1 to 2 % of the time); 61 % of the slots taken, the integer pipe 55 % busy. Columns by 8 keep 128 registers and four CTAs on an SM, by 16 (more
// than 8 columns) they share a page's unpacking. Codes turned into BF16 operands first took 204 us, as subnormal ones 136, sums of p lo as a product 109.
constexpr int KV4_WARPS = 4, KV4_SLOTS = 2;      // (a warp for every group of a head at least)
constexpr int KV4_KEPT = 4;                      // binades that a page's values may lie below the power of two that a warp has for them
template <int D, int NT>
constexpr int kv4_smem() {
  const int ring = KV4_WARPS * (KV4_SLOTS * kv4_page_bytes(D) + KV4_PAGE * D / 8), merge = (KV4_WARPS * (D + D / 32 + 2) + D + 2) * NT * 8 * 4;
  return ring > merge ? ring : merge;
}

template <int D, int NT>
__global__ void __launch_bounds__(32 * KV4_WARPS, NT == 1 ? 4 : 2)
kv4_rows_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ kpages, const uint8_t* __restrict__ vpages, const int* __restrict__ block_table,
                const int* __restrict__ q_start, const int* __restrict__ q_lens, const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out,
                float* __restrict__ part_o, float2* __restrict__ part_ml, int rows, int nq, int hq, int hkv, long long ldq, long long ldo, int max_blocks, int num_blocks,
                int nsplit, uint32_t per_group, float scale_log2, int* status) {
  constexpr int NG = D / 32, PB = kv4_page_bytes(D), ROW = D / 2, STAT = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[KV4_WARPS][KV4_SLOTS];
  __shared__ uint4 sq[NT][NG][32];
  __shared__ float ssum[NT][NG][8];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x < KV4_WARPS * KV4_SLOTS) mbar_init(&full[threadIdx.x / KV4_SLOTS][threadIdx.x % KV4_SLOTS], 1);
  mbar_fence_init();
  __syncthreads();
  pdl_wait();
  const int split = blockIdx.x, kvh = blockIdx.y % hkv, ct = blockIdx.y / hkv, b = blockIdx.z;
  const int G = hq / hkv;
  auto group_of = [&](int c) -> int { return per_group ? (int)__umulhi((uint32_t)c, per_group) : c; };      // c / G
  const int n = q_lens ? q_lens[b] : nq, row0 = q_start ? q_start[b] : b * nq;
  int ctx = ctx_lens[b];
  if (n > 0 && (n > nq || row0 < 0 || n > rows - row0)) {       // rows that the call does not have
    if (threadIdx.x == 0) set_status(status, KID_ATTN_DECODE, FF_ERR_BOUNDS, b, row0);
    return;
  }
  const int columns = n * G - ct * NT * 8;                      // of this CTA and behind it
  if (columns <= 0) return;
  // queries of this thread's column of B fragments (column g of every 8): 8 elements of each group
  uint4 qv[NT][NG];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int c = ct * NT * 8 + nt * 8 + g;
    const bool live = nt * 8 + g < columns;
    const int qi = live ? group_of(c) : 0;
    const __nv_bfloat16* src = q + (size_t)(row0 + qi) * ldq + (size_t)(kvh * G + (live ? c - qi * G : 0)) * D;
#pragma unroll
    for (int j = 0; j < NG; ++j) qv[nt][j] = live ? *reinterpret_cast<const uint4*>(src + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
  }
  if (ctx > max_blocks * KV4_PAGE) {                            // more keys than the table has pages
    if (threadIdx.x == 0) set_status(status, KID_ATTN_DECODE, FF_ERR_BOUNDS, b, ctx);
    ctx = max_blocks * KV4_PAGE;
  }
  // keys that the last of this CTA's columns sees; its pages are shared evenly by the splits and, one after the other, by the warps
  const int seen = min(ctx, ctx - n + group_of(ct * NT * 8 + min(columns, NT * 8) - 1) + 1);
  const int pages = (max(seen, 0) + KV4_PAGE - 1) / KV4_PAGE;
  const int per = max((pages + nsplit - 1) / nsplit, KV4_WARPS);       // a page for every warp at least: a launch for long contexts may meet a short one
  const int p0 = split * per + warp, p1 = min(pages, split * per + per);
  const int mine = p1 > p0 ? (p1 - p0 + KV4_WARPS - 1) / KV4_WARPS : 0;

  // numbers of this warp's pages: a lane each, 32 ahead
  bool bad = false;
  auto numbers = [&](int first) -> int {
    const int p = p0 + (first + lane) * KV4_WARPS;
    if (p >= p1) return 0;
    const int blk = block_table[(size_t)b * max_blocks + p];
    if (blk < 0 || blk >= num_blocks) { bad = true; return 0; }
    return blk;
  };
  int ids = numbers(0), ids_next = mine > 32 ? numbers(32) : 0;
  uint8_t* const ring = smem + warp * (KV4_SLOTS * PB);
  auto issue = [&](int i) {                                     // item i: keys (even) or values of page i / 2; the whole warp
    const int blk = __shfl_sync(0xffffffffu, ids, (i >> 1) & 31);
    if (lane == 0) {
      const int slot = i % KV4_SLOTS;
      mbar_expect_tx(&full[warp][slot], PB);
      kv4_bulk_load(ring + slot * PB, ((i & 1) ? vpages : kpages) + ((size_t)blk * hkv + kvh) * PB, PB, &full[warp][slot]);
    }
  };
#pragma unroll
  for (int i = 0; i < KV4_SLOTS; ++i)
    if (i < 2 * mine) issue(i);

  // B fragments of the queries: the warps make those of a group each and share them; in registers they are only while a page's keys are multiplied
  uint32_t qb[NT][2];
  float cf[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint32_t w[4] = {qv[nt][j].x, qv[nt][j].y, qv[nt][j].z, qv[nt][j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(kv4_low(w[i])), fabsf(kv4_high(w[i]))));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1)); most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^(14 - exponent) of the column's greatest element, and 2^24 over it (zero columns: any; the exponents are kept where both are normal numbers)
    const int ex = min(max((int)(__float_as_uint(most) >> 23), 20), 244);
    const float gain = __uint_as_float((uint32_t)(min(254 + 14 - ex, 254)) << 23), back = __uint_as_float((uint32_t)(254 - min(254 + 14 - ex, 254) + 24) << 23);
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      if (j != warp) continue;
      const uint32_t w[4] = {qv[nt][j].x, qv[nt][j].y, qv[nt][j].z, qv[nt][j].w};
      uint32_t f[4];
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = kv4_low(w[i]) * gain, y = kv4_high(w[i]) * gain;
        s += x + y;
        f[i] = (i & 1) ? kv4_f16x2(x * 0.0625f, y * 0.0625f) : kv4_f16x2(x, y);
      }
      s += __shfl_xor_sync(0xffffffffu, s, 1); s += __shfl_xor_sync(0xffffffffu, s, 2);
      sq[nt][j][lane] = make_uint4(f[0], f[1], f[2], f[3]);
      if (t == 0) ssum[nt][j][g] = s * 5.9604644775390625e-8f;                       // 2^-24
    }
    const float f = fmaxf(scale_log2 * back, 1.1754944e-38f);   // (times minus infinity it has to be that)
    cf[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);             // column 2 t is held by lanes of g = 2 t
    cf[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
    for (int e = 0; e < 2; ++e) lim[nt][e] = nt * 8 + 2 * t + e < columns ? ctx - n + group_of(ct * NT * 8 + nt * 8 + 2 * t + e) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // sum(q) of the group that this lane has in the product with lo, in three parts
    const float s = t < NG ? ssum[nt][t & (NG - 1)][g] : 0.f, a = __bfloat162float(__float2bfloat16(s)), c = __bfloat162float(__float2bfloat16(s - a));
    qb[nt][0] = pack_bf16x2(a, c); qb[nt][1] = pack_bf16x2(s - a - c, 0.f);
  }
  const int all = ctx - n + group_of(ct * NT * 8);                    // keys up to here are seen by every column

  float o[NT][NG][2][4], ol[NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = KV4_NONE; l[nt][0] = l[nt][1] = 0.f;
    ol[nt][0] = ol[nt][1] = ol[nt][2] = ol[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
#pragma unroll
      for (int a = 0; a < 2; ++a) o[nt][j][a][0] = o[nt][j][a][1] = o[nt][j][a][2] = o[nt][j][a][3] = 0.f;
    }
  }

  // exponent field of the power of two that this warp's values are divided by (what O holds is divided by it too), and its greatest so far
  int ref = KV4_LEAST, top = KV4_LEAST;
  const uint32_t stats_at = smem_u32(smem + KV4_WARPS * KV4_SLOTS * PB) + warp * (KV4_PAGE * STAT);
  // row r of a 16-key tile is key 4 (r / 2) + r % 2, two more from r = 8 on: a thread's four columns of P^T are then its keys 4 t .. 4 t + 3
  const int kg = 4 * (g >> 1) + (g & 1);
  const uint32_t ring_at = smem_u32(ring);
  bool ok = true;
  RingPos pos;
  for (int w = 0; w < mine; ++w) {
    const int p = p0 + w * KV4_WARPS;
    const bool whole = p * KV4_PAGE + KV4_PAGE - 1 <= all;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][pos.s], pos.ph, nullptr, status, KID_ATTN_DECODE, 41));      // (lanes give up together: those that went on would wait for the others)
    if (!ok) break;
    float s[4][NT][4];
    {
      const uint32_t sk = ring_at + pos.s * PB;
      uint32_t qf[NT][NG][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NG; ++j) kv4_lds(smem_u32(&sq[nt][j][lane]), qf[nt][j][0][0], qf[nt][j][0][1], qf[nt][j][1][0], qf[nt][j][1][1]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        uint32_t kw[2][NG], ks[2][NG], la[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = mt * 16 + kg + 2 * r;
          kv4_words<NG>(kw[r], sk + key * ROW + t * (D / 8));
          kv4_words<NG>(ks[r], sk + kv4_code_bytes(D) + key * STAT);
          // lo of group t, twice (with two groups the other lanes' queries are zero, but what they would read may be no number)
          la[r] = 0u;
          if (NG == 4 || t < NG) {
            uint32_t st;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(st) : "r"(sk + kv4_code_bytes(D) + key * STAT + 4 * t) : "memory");
            la[r] = kv4_prmt(st, st, 0x3232u);
          }
        }
        const uint32_t al[4] = {la[0], la[1], la[0], la[1]};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
          ms_mma(s[mt][nt], al, qb[nt][0], qb[nt][1]);
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
          uint32_t w0 = kw[0][j], w1 = kw[1][j];
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const uint32_t a[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) kv4_mma(acc[nt], a, qf[nt][j][k2][0], qf[nt][j][k2][1]);
            w0 >>= 8; w1 >>= 8;
          }
          const float f0 = kv4_low(ks[0][j]), f1 = kv4_low(ks[1][j]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[mt][nt][0] = fmaf(f0, acc[nt][0], s[mt][nt][0]);
            s[mt][nt][1] = fmaf(f0, acc[nt][1], s[mt][nt][1]);
            s[mt][nt][2] = fmaf(f1, acc[nt][2], s[mt][nt][2]);
            s[mt][nt][3] = fmaf(f1, acc[nt][3], s[mt][nt][3]);
          }
        }
      }
    }
    __syncwarp();                                               // the slot is read
    if (w + 1 < mine) {                                         // keys of the next page
      if (((w + 1) & 31) == 0) { ids = ids_next; ids_next = numbers(w + 33); }
      issue(2 * w + 2);
    }
    pos.next(KV4_SLOTS);
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (p * KV4_PAGE + mt * 16 + kg + 2 * (r >> 1) > lim[nt][r & 1]) s[mt][nt][r] = -INFINITY;
      __syncwarp();                                             // (a branch of its own: the selects are not worth their place in every other page)
    }
    // running maxima of columns 2 t and 2 t + 1, weights times 2^7 (their sum has the factor too)
    float alpha[NT][2];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) mx = fmaxf(mx, s[mt][nt][2 * r + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][e], mx * cf[nt][e]);
        alpha[nt][e] = kv4_ex2(m[nt][e] - mn);
        moved = moved || mn != m[nt][e];
        m[nt][e] = mn;
        const float off = 7.0f - mn;
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& v = s[mt][nt][2 * r + e];
            v = kv4_ex2(fmaf(v, cf[nt][e], off));
            sum += v;
          }
        l[nt][e] = fmaf(l[nt][e], alpha[nt][e], sum);
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          ol[nt][e] *= alpha[nt][e];
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int a = 0; a < 2; ++a) { o[nt][j][a][e] *= alpha[nt][e]; o[nt][j][a][2 + e] *= alpha[nt][e]; }
        }
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][pos.s], pos.ph, nullptr, status, KID_ATTN_DECODE, 42));
    if (!ok) break;
    const uint32_t sv = ring_at + pos.s * PB;
    {
      // (scale, lo) of the page times 2^7 over the power of two: exact in BF16, and 2^8 at most
      uint32_t st[NG / 2][4], most = 0u;
#pragma unroll
      for (int i = 0; i < NG / 2; ++i) {
        kv4_lds(sv + kv4_code_bytes(D) + 16 * (lane + 32 * i), st[i][0], st[i][1], st[i][2], st[i][3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // tokens behind the sequence: whatever the page holds there is no number, and 0 times it would not be 0
          if (p * KV4_PAGE + KV4_PAGE > ctx && p * KV4_PAGE + (4 * (lane + 32 * i) + k) / NG >= ctx) st[i][k] = 0u;
          most = kv4_maxabs2(most, st[i][k]);
        }
      }
      const int ex = max((int)(kv4_warp_max(max(most & 0x7fffu, most >> 16 & 0x7fffu)) >> 7), KV4_LEAST);
      if (ex > ref || ex + KV4_KEPT < ref) {                    // (for all lanes)
        top = max(top, ex);
        const int next = max(ex, top - KV4_SPAN);
        const float f = __uint_as_float((uint32_t)(127 + ref - next) << 23);
        ref = next;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ol[nt][e] *= f;
#pragma unroll
            for (int j = 0; j < NG; ++j) { o[nt][j][0][e] *= f; o[nt][j][1][e] *= f; }
          }
      }
      const uint32_t by = (uint32_t)(261 - ref) * 0x00800080u;
#pragma unroll
      for (int i = 0; i < NG / 2; ++i)
        kv4_sts(stats_at + 16 * (lane + 32 * i), kv4_mul2(st[i][0], by), kv4_mul2(st[i][1], by), kv4_mul2(st[i][2], by), kv4_mul2(st[i][3], by));
      __syncwarp();
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t vs[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = mt * 16 + kg + 2 * r;
        kv4_words<NG>(vs[r], stats_at + key * STAT);
      }
      {
        // rows of A: lo of group g % NG (rows 8 .. 15: nothing)
        uint32_t st[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(st[i]) : "r"(stats_at + (mt * 16 + 4 * t + i) * STAT + 4 * (g & (NG - 1))) : "memory");
        const uint32_t a[4] = {kv4_f16x2(kv4_high(st[0]), kv4_high(st[1])), 0u, kv4_f16x2(kv4_high(st[2]), kv4_high(st[3])), 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          kv4_mma(ol[nt], a, kv4_transpose(kv4_f16x2(s[mt][nt][0], s[mt][nt][1])), kv4_transpose(kv4_f16x2(s[mt][nt][2], s[mt][nt][3])));
      }
      uint32_t vw[4][NG / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = sv + kv4_value_at<D>(mt * 16 + 4 * t + i, g, 0);
        if constexpr (NG == 4) kv4_lds(at, vw[i][0], vw[i][1]);
        else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(vw[i][0]) : "r"(at) : "memory");
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        uint32_t x01 = kv4_prmt(vw[0][j / 2], vw[1][j / 2], sel), x23 = kv4_prmt(vw[2][j / 2], vw[3][j / 2], sel);
        const float f0 = kv4_low(vs[0][j]), f1 = kv4_low(vs[1][j]);
        uint32_t bf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf[nt][0] = kv4_transpose(kv4_f16x2(s[mt][nt][0] * f0, s[mt][nt][1] * f0));
          bf[nt][1] = kv4_transpose(kv4_f16x2(s[mt][nt][2] * f1, s[mt][nt][3] * f1));
        }
#pragma unroll
        for (int a2 = 0; a2 < 2; ++a2) {
          const uint32_t a[4] = {x01 & 0x000f000fu, x01 & 0x00f000f0u, x23 & 0x000f000fu, x23 & 0x00f000f0u};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) kv4_mma(o[nt][j][a2], a, bf[nt][0], bf[nt][1]);
          x01 >>= 8; x23 >>= 8;
        }
      }
    }
    __syncwarp();
    if (w + 1 < mine) issue(2 * w + 3);                         // its values
    pos.next(KV4_SLOTS);
  }
  if (bad) set_status(status, KID_ATTN_DECODE, FF_ERR_BOUNDS, b, split);
  if (!ok) {                                                    // a copy that never came: give those in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();                                              // the rings are free

  float* const so = reinterpret_cast<float*>(smem);             // [warp][column][D], then [warp][column][2], [warp][column][NG]; this CTA's [column][D], [column][2]
  float* const sml = so + KV4_WARPS * NT * 8 * D;
  float* const sol = sml + KV4_WARPS * NT * 8 * 2;
  float* const mo = sol + KV4_WARPS * NT * 8 * NG;
  float* const mml = mo + NT * 8 * D;
  const bool cluster = nsplit > 1 && part_o == nullptr;         // the splits are a cluster and join in shared memory
  // the powers of two out of O: of the values, and of the codes at bits 0 .. 3 and 4 .. 7
  const float of_lo = __uint_as_float((uint32_t)(ref - 7) << 23), of_even = __uint_as_float((uint32_t)(ref + 17) << 23), of_odd = __uint_as_float((uint32_t)(ref + 13) << 23);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = nt * 8 + 2 * t + e;
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4); l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      if (g == 0) { sml[(warp * NT * 8 + col) * 2] = m[nt][e]; sml[(warp * NT * 8 + col) * 2 + 1] = l[nt][e]; }
      if (g < NG) sol[(warp * NT * 8 + col) * NG + g] = ol[nt][e] * of_lo;
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)                             // nibble i of lane g's unit: element 32 j + 8 (g / 2) + 2 i + g % 2
          so[(warp * NT * 8 + col) * D + 32 * j + 8 * (g >> 1) + 2 * i + (g & 1)] = o[nt][j][i >> 1][2 * (i & 1) + e] * ((i & 1) ? of_odd : of_even);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < min(columns, NT * 8) * D; i += 32 * KV4_WARPS) {
    const int col = i / D, d = i - col * D;
    float M = KV4_NONE, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < KV4_WARPS; ++w) M = fmaxf(M, sml[(w * NT * 8 + col) * 2]);
#pragma unroll
    for (int w = 0; w < KV4_WARPS; ++w) {
      const float sc = exp2f(sml[(w * NT * 8 + col) * 2] - M);
      L += sml[(w * NT * 8 + col) * 2 + 1] * sc;
      acc += (so[(w * NT * 8 + col) * D + d] + sol[(w * NT * 8 + col) * NG + (d >> 5)]) * sc;
    }
    const int c = ct * NT * 8 + col, qi = group_of(c), head = kvh * G + c - qi * G;
    if (nsplit == 1) {
      out[(size_t)(row0 + qi) * ldo + (size_t)head * D + d] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
    } else if (cluster) {
      mo[i] = acc;
      if (d == 0) { mml[2 * col] = M; mml[2 * col + 1] = L; }
    } else {
      const size_t pr = ((size_t)(row0 + qi) * hq + head) * nsplit + split;
      part_o[pr * D + d] = acc;
      if (d == 0) part_ml[pr] = make_float2(M, L);
    }
  }
  if (cluster) {
    cluster_sync_all();
    for (int i = split * 32 * KV4_WARPS + threadIdx.x; i < min(columns, NT * 8) * D; i += nsplit * 32 * KV4_WARPS) {
      const int col = i / D, d = i - col * D;
      float2 ml[8];
      float M = KV4_NONE, L = 0.f, acc = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < nsplit) { ml[r] = kv4_peer2(mml + 2 * col, r); M = fmaxf(M, ml[r].x); }
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < nsplit) {
          const float sc = kv4_ex2(ml[r].x - M);
          L = fmaf(ml[r].y, sc, L);
          acc = fmaf(kv4_peer(mo + i, r), sc, acc);
        }
      const int c = ct * NT * 8 + col, qi = group_of(c), head = kvh * G + c - qi * G;
      out[(size_t)(row0 + qi) * ldo + (size_t)head * D + d] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
    }
    cluster_sync_all();                                         // no CTA leaves while its shared memory is read
  }
}

// More than eight splits of one (row, head) joined: four warps take every fourth split, a lane D / 32 elements, four splits on their way at once (one after the
// other, 74 splits of a single sequence took as long as the attention itself).
template <int D>
__global__ void __launch_bounds__(128)
kv4_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, __nv_bfloat16* __restrict__ out, int hq, long long ldo, int nsplit) {
  constexpr int E = D / 32;
  __shared__ float sacc[4][D];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x / hq, head = blockIdx.x - row * hq;
  const size_t pr = ((size_t)row * hq + head) * nsplit;
  float2 ml[4];                                                 // of splits lane, lane + 32, ... (at most 128)
  float M = KV4_NONE, L = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ml[i] = lane + 32 * i < nsplit ? part_ml[pr + lane + 32 * i] : make_float2(KV4_NONE, 0.f);
    M = fmaxf(M, ml[i].x);
  }
  M = warp_max(M);
#pragma unroll
  for (int i = 0; i < 4; ++i) { ml[i].x = kv4_ex2(ml[i].x - M); L = fmaf(ml[i].y, ml[i].x, L); }
  L = warp_sum(L);
  float acc[E];
#pragma unroll
  for (int k = 0; k < E; ++k) acc[k] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    for (int s = 32 * i + warp; s < min(nsplit, 32 * i + 32); s += 16) {
      float v[4][E], sc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = s + 4 * u;
        sc[u] = __shfl_sync(0xffffffffu, ml[i].x, at & 31);
        if (at >= min(nsplit, 32 * i + 32)) sc[u] = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) v[u][k] = sc[u] != 0.f ? part_o[(pr + at) * D + lane + 32 * k] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] = fmaf(v[u][k], sc[u], acc[k]);
    }
#pragma unroll
  for (int k = 0; k < E; ++k) sacc[warp][lane + 32 * k] = acc[k];
  __syncthreads();
  const int d = threadIdx.x;
  if (d < D) {
    const float o = (sacc[0][d] + sacc[1][d]) + (sacc[2][d] + sacc[3][d]);
    out[(size_t)row * ldo + (size_t)head * D + d] = __float2bfloat16(L == 0.f ? 0.f : o / L);
  }
}

}  // namespace ff
using namespace ff;

// Splits that ff_kv4_attn_rows takes for such a launch, and the floats of scratch it needs for them (none up to eight).
FF_EXPORT int ff_kv4_attn_plan(int batch, int hq, int hkv, int nq, int dim, int max_ctx, long long* floats) {
  const int columns = nq * (hq / hkv), pages = (max_ctx + KV4_PAGE - 1) / KV4_PAGE;
  const long long ctas = (long long)batch * hkv * (columns > 8 ? (columns + 15) / 16 : 1);
  long long nsplit = ((columns > 8 ? 2ll : 4ll) * sm_count()) / ctas;
  const long long most = (pages + KV4_WARPS - 1) / KV4_WARPS;
  if (nsplit > most) nsplit = most;
  if (nsplit > 128) nsplit = 128;
  if (nsplit < 1) nsplit = 1;
  if (floats) *floats = nsplit > 8 ? (long long)batch * nq * hq * nsplit * (dim + 2) : 0;
  return (int)nsplit;
}

// q rows [rows, ldq] with head h at column h dim; sequence b has rows q_start[b] .. + q_lens[b], or nq rows from b nq on where those are null (only then may
// there be more than eight splits); ctx_lens[b] keys are seen by the last of them. Rows of no keys are zero.
FF_EXPORT int ff_kv4_attn_rows(const void* q, const void* kpages, const void* vpages, const int* block_table, const int* q_start, const int* q_lens,
                               const int* ctx_lens, void* out, float* scratch, int batch, int rows, int nq, int hq, int hkv, int dim, long long ldq,
                               long long ldo, int max_blocks, int num_blocks, int nsplit, float scale, int* status, cudaStream_t s) {
  if (batch <= 0 || batch > 65535 || rows <= 0 || nq <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || (dim != 64 && dim != 128) || max_blocks <= 0 || num_blocks <= 0) return FF_HOST_BAD_SHAPE;
  if (!(scale > 0.f) || nsplit < 1 || nsplit > 128 || (q_start == nullptr) != (q_lens == nullptr) || (nsplit > 8 && (scratch == nullptr || q_start != nullptr))) return FF_HOST_BAD_SHAPE;
  if (ldq % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kpages) | reinterpret_cast<uintptr_t>(vpages)) & 15)) return FF_HOST_BAD_ALIGN;
  const int columns = nq * (hq / hkv);
  const bool wide = columns > 8;
  const long long tiles = (long long)hkv * (wide ? (columns + 15) / 16 : 1);
  if (tiles > 65535) return FF_HOST_TOO_LARGE;
  auto kern = dim == 128 ? (wide ? kv4_rows_kernel<128, 2> : kv4_rows_kernel<128, 1>) : (wide ? kv4_rows_kernel<64, 2> : kv4_rows_kernel<64, 1>);
  const int bytes = dim == 128 ? (wide ? kv4_smem<128, 2>() : kv4_smem<128, 1>()) : (wide ? kv4_smem<64, 2>() : kv4_smem<64, 1>());
  if (int r = opt_in_smem(kern, bytes)) return r;
  if (q_start == nullptr && (long long)batch * nq != rows) return FF_HOST_BAD_SHAPE;
  float2* ml = nsplit > 8 ? reinterpret_cast<float2*>(scratch + (long long)rows * hq * nsplit * dim) : nullptr;
  if (int r = launch_pdl(kern, dim3(nsplit, (unsigned)tiles, batch), dim3(32 * KV4_WARPS), bytes, s, nsplit <= 8 ? nsplit : 0, (const __nv_bfloat16*)q, (const uint8_t*)kpages,
                         (const uint8_t*)vpages, block_table, q_start, q_lens, ctx_lens, (__nv_bfloat16*)out, nsplit > 8 ? scratch : (float*)nullptr, ml, rows, nq, hq, hkv, ldq, ldo, max_blocks,
                         num_blocks, nsplit, hq == hkv ? 0u : (uint32_t)((0x100000000ull + hq / hkv - 1) / (hq / hkv)), scale * 1.4426950408889634f, status)) return r;
  if (nsplit <= 8) return FF_HOST_OK;
  if ((long long)rows * hq > 0x7fffffffll) return FF_HOST_TOO_LARGE;
  return launch_pdl(dim == 128 ? kv4_merge_kernel<128> : kv4_merge_kernel<64>, dim3((unsigned)(rows * hq)), dim3(128), 0, s, 0, (const float*)scratch, (const float2*)ml,
                    (__nv_bfloat16*)out, hq, ldo, nsplit);
}
