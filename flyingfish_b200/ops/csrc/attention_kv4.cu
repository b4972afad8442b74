// Attention over the 4-bit key / value cache (layout and format: kv4.cuh).
#include "kv4.cuh"
#include "host_util.h"
#include "mma_sync.cuh"

namespace ff {

constexpr float KV4_NEG = -3.0e38f;

__device__ __forceinline__ uint32_t kv4_prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// the 8 x 8 matrix of 16-bit elements that the warp's registers hold by rows, transposed
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// nibbles at bits 4 i and 4 i + 16 as BF16 numbers: 128 + n is a BF16 number with n in its last bits, the difference is exact
__device__ __forceinline__ uint32_t kv4_codes(uint32_t w, int shift) {
  uint32_t v = ((w >> shift) & 0x000f000fu) | 0x43004300u;
  const uint32_t m = 0xc300c300u;
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(m));
  return r;
}
__device__ __forceinline__ void kv4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Rows of queries, a few per sequence (one in a decode step): the rows of one sequence times the query heads of one kv head are the columns of
//   S^T [keys x columns] = K Q^T        O^T [elements x columns] = V^T P^T
// so that the cache is the 16-row operand of mma.sync m16n8k16 and 8 columns are enough to fill an instruction. Codes 0 .. 15 go into the products as
// they are; with the groups j of 32 elements
//   S = sum_j scale_j (q_j . n_j) + lo_j sum(q_j)          O_j = sum_k (p_k scale_kj) n_kj + sum_k p_k lo_kj
// scale and lo of the keys meet the scores in FP32, those of the values the probabilities (p scale is what is rounded to BF16).
// A CTA has NT x 8 columns and a range of pages; every warp takes pages of its own, with its own ring of stages that bulk copies fill, its own running
// maximum, sum and O. The warps' results meet in shared memory, those of several CTAs (splits) in kv4_merge_kernel.
constexpr int KV4_WARPS = 4, KV4_STAGES = 2;
template <int D, int NT>
constexpr int kv4_smem() {
  const int ring = KV4_WARPS * KV4_STAGES * 2 * kv4_page_bytes(D), merge = KV4_WARPS * NT * 8 * (D + 2) * 4;
  return ring > merge ? ring : merge;
}

template <int D, int NT>
__global__ void __launch_bounds__(32 * KV4_WARPS)
kv4_rows_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ kpages, const uint8_t* __restrict__ vpages, const int* __restrict__ block_table,
                const int* __restrict__ q_start, const int* __restrict__ q_lens, const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out,
                float* __restrict__ part_o, float2* __restrict__ part_ml, int nq, int hq, int hkv, long long ldq, long long ldo, int max_blocks, int num_blocks,
                int nsplit, float scale_log2, int* status) {
  constexpr int NG = D / 32, PB = kv4_page_bytes(D), ROW = D / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[KV4_WARPS][KV4_STAGES];
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x, kvh = blockIdx.y % hkv, ct = blockIdx.y / hkv, b = blockIdx.z;
  const int G = hq / hkv;
  const int n = q_lens ? q_lens[b] : nq, row0 = q_start ? q_start[b] : b * nq;
  const int columns = n * G - ct * NT * 8;                      // of this CTA and behind it
  if (columns <= 0) return;
  int ctx = ctx_lens[b];
  if (ctx > max_blocks * KV4_PAGE) {                            // more keys than the table has pages
    if (threadIdx.x == 0) set_status(status, KID_ATTN_DECODE, FF_ERR_BOUNDS, b, ctx);
    ctx = max_blocks * KV4_PAGE;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // keys that the last of this CTA's columns sees
  const int seen = min(ctx, ctx - n + (ct * NT * 8 + min(columns, NT * 8) - 1) / G + 1);
  const int pages = (max(seen, 0) + KV4_PAGE - 1) / KV4_PAGE;
  const int per = (pages + nsplit - 1) / nsplit;
  const int p0 = split * per, p1 = min(pages, p0 + per);
  if (threadIdx.x < KV4_WARPS * KV4_STAGES) mbar_init(&full[threadIdx.x / KV4_STAGES][threadIdx.x % KV4_STAGES], 1);
  mbar_fence_init();
  __syncthreads();

  bool bad = false;
  uint8_t* const ring = smem + warp * (KV4_STAGES * 2 * PB);
  auto issue = [&](int p, int st) {
    int blk = block_table[(size_t)b * max_blocks + p];
    if (blk < 0 || blk >= num_blocks) { bad = true; blk = 0; }
    const size_t at = ((size_t)blk * hkv + kvh) * PB;
    mbar_expect_tx(&full[warp][st], 2 * PB);
    kv4_bulk_load(ring + st * 2 * PB, kpages + at, PB, &full[warp][st]);
    kv4_bulk_load(ring + st * 2 * PB + PB, vpages + at, PB, &full[warp][st]);
  };
  if (lane == 0)
    for (int i = 0; i < KV4_STAGES; ++i)
      if (p0 + warp + i * KV4_WARPS < p1) issue(p0 + warp + i * KV4_WARPS, i);

  // queries of this thread's column of B fragments (column g of every 8), sums of the groups of columns 2 t and 2 t + 1
  uint32_t qf[NT][NG][2][2];
  float qs[NT][NG][2];
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int c = ct * NT * 8 + nt * 8 + g;
    const bool live = nt * 8 + g < columns;
    const __nv_bfloat16* src = q + (size_t)(row0 + (live ? c / G : 0)) * ldq + (size_t)(kvh * G + (live ? c % G : 0)) * D;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (live) v = *reinterpret_cast<const uint4*>(src + 32 * j + 8 * t);
      qf[nt][j][0][0] = v.x; qf[nt][j][0][1] = v.y; qf[nt][j][1][0] = v.z; qf[nt][j][1][1] = v.w;
      const float2 a = unpack_bf16x2(v.x), e = unpack_bf16x2(v.y), f = unpack_bf16x2(v.z), h = unpack_bf16x2(v.w);
      float s = ((a.x + a.y) + (e.x + e.y)) + ((f.x + f.y) + (h.x + h.y));
      s += __shfl_xor_sync(0xffffffffu, s, 1); s += __shfl_xor_sync(0xffffffffu, s, 2);
      qs[nt][j][0] = __shfl_sync(0xffffffffu, s, 8 * t);        // column 2 t is held by lanes of g = 2 t
      qs[nt][j][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) lim[nt][e] = nt * 8 + 2 * t + e < columns ? ctx - n + (ct * NT * 8 + nt * 8 + 2 * t + e) / G : -1;
  }
  const int all = ctx - n + ct * NT * 8 / G;                    // keys up to here are seen by every column

  float o[NT][NG][2][4], ol[NT][NG][2], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = KV4_NEG; l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      ol[nt][j][0] = ol[nt][j][1] = 0.f;
#pragma unroll
      for (int a = 0; a < 2; ++a) o[nt][j][a][0] = o[nt][j][a][1] = o[nt][j][a][2] = o[nt][j][a][3] = 0.f;
    }
  }

  bool ok = true;
  int it = 0;
  for (int p = p0 + warp; p < p1; p += KV4_WARPS, ++it) {
    const int st = it % KV4_STAGES;
    if (!mbar_wait(&full[warp][st], (it / KV4_STAGES) & 1, nullptr, status, KID_ATTN_DECODE, 41)) { ok = false; break; }
    const uint8_t* sk = ring + st * 2 * PB;
    const uint8_t* sv = sk + PB;
    const bool whole = p * KV4_PAGE + KV4_PAGE - 1 <= all;
    float s[4][NT][4];
    // row r of a 16-key tile is key 4 (r / 2) + r % 2, two more from r = 8 on: a thread's four columns of P^T are then its keys 4 t .. 4 t + 3
    const int kg = 4 * (g >> 1) + (g & 1);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t kw[2][NG];
      uint32_t ks[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = mt * 16 + kg + 2 * r;
        if (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(sk + key * ROW + t * 16);
          kw[r][0] = v.x; kw[r][1] = v.y; kw[r][NG - 2] = v.z; kw[r][NG - 1] = v.w;
          const uint4 f = *reinterpret_cast<const uint4*>(sk + kv4_code_bytes(D) + key * 16);
          ks[r][0] = f.x; ks[r][1] = f.y; ks[r][NG - 2] = f.z; ks[r][NG - 1] = f.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(sk + key * ROW + t * 8);
          kw[r][0] = v.x; kw[r][1] = v.y;
          const uint2 f = *reinterpret_cast<const uint2*>(sk + kv4_code_bytes(D) + key * 8);
          ks[r][0] = f.x; ks[r][1] = f.y;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          const uint32_t a[4] = {kv4_codes(kw[0][j], 8 * k2), kv4_codes(kw[1][j], 8 * k2), kv4_codes(kw[0][j], 8 * k2 + 4), kv4_codes(kw[1][j], 8 * k2 + 4)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) ms_mma(acc[nt], a, qf[nt][j][k2][0], qf[nt][j][k2][1]);
        }
        const float2 f0 = unpack_bf16x2(ks[0][j]), f1 = unpack_bf16x2(ks[1][j]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[mt][nt][0] = fmaf(f0.x, acc[nt][0], fmaf(f0.y, qs[nt][j][0], s[mt][nt][0]));
          s[mt][nt][1] = fmaf(f0.x, acc[nt][1], fmaf(f0.y, qs[nt][j][1], s[mt][nt][1]));
          s[mt][nt][2] = fmaf(f1.x, acc[nt][2], fmaf(f1.y, qs[nt][j][0], s[mt][nt][2]));
          s[mt][nt][3] = fmaf(f1.x, acc[nt][3], fmaf(f1.y, qs[nt][j][1], s[mt][nt][3]));
        }
      }
    }
    // masks, running maxima of columns 2 t and 2 t + 1 (in raw units: the scale is positive)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = KV4_NEG;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& v = s[mt][nt][2 * r + e];
            v *= scale_log2;
            if (!whole && p * KV4_PAGE + mt * 16 + kg + 2 * r > lim[nt][e]) v = KV4_NEG;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][e], mx), alpha = exp2f(m[nt][e] - mn);
        m[nt][e] = mn;
        l[nt][e] *= alpha;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          ol[nt][j][e] *= alpha;
#pragma unroll
          for (int a = 0; a < 2; ++a) { o[nt][j][a][e] *= alpha; o[nt][j][a][2 + e] *= alpha; }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float& v = s[mt][nt][2 * r + e];
            v = v <= KV4_NEG ? 0.f : exp2f(v - mn);
            l[nt][e] += v;
          }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t vs[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = mt * 16 + kg + 2 * r;
        if (NG == 4) {
          const uint4 f = *reinterpret_cast<const uint4*>(sv + kv4_code_bytes(D) + key * 16);
          vs[r][0] = f.x; vs[r][1] = f.y; vs[r][NG - 2] = f.z; vs[r][NG - 1] = f.w;
        } else {
          const uint2 f = *reinterpret_cast<const uint2*>(sv + kv4_code_bytes(D) + key * 8);
          vs[r][0] = f.x; vs[r][1] = f.y;
        }
        // tokens behind the sequence: whatever a page holds there (their probabilities are 0)
        if (!whole && p * KV4_PAGE + key >= ctx) {
#pragma unroll
          for (int j = 0; j < NG; ++j) vs[r][j] = 0u;
        }
      }
      uint32_t vw[4][NG / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* at = sv + kv4_value_at<D>(mt * 16 + 4 * t + i, g, 0);
        if (NG == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(at);
          vw[i][0] = v.x; vw[i][NG / 2 - 1] = v.y;
        } else {
          vw[i][0] = *reinterpret_cast<const uint32_t*>(at);
        }
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        const uint32_t x01 = kv4_prmt(vw[0][j / 2], vw[1][j / 2], sel), x23 = kv4_prmt(vw[2][j / 2], vw[3][j / 2], sel);
        const float2 f0 = unpack_bf16x2(vs[0][j]), f1 = unpack_bf16x2(vs[1][j]);
        uint32_t bf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf[nt][0] = kv4_transpose(pack_bf16x2(s[mt][nt][0] * f0.x, s[mt][nt][1] * f0.x));
          bf[nt][1] = kv4_transpose(pack_bf16x2(s[mt][nt][2] * f1.x, s[mt][nt][3] * f1.x));
          ol[nt][j][0] = fmaf(s[mt][nt][0], f0.y, fmaf(s[mt][nt][2], f1.y, ol[nt][j][0]));
          ol[nt][j][1] = fmaf(s[mt][nt][1], f0.y, fmaf(s[mt][nt][3], f1.y, ol[nt][j][1]));
        }
#pragma unroll
        for (int a2 = 0; a2 < 2; ++a2) {
          const uint32_t a[4] = {kv4_codes(x01, 8 * a2), kv4_codes(x01, 8 * a2 + 4), kv4_codes(x23, 8 * a2), kv4_codes(x23, 8 * a2 + 4)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) ms_mma(o[nt][j][a2], a, bf[nt][0], bf[nt][1]);
        }
      }
    }
    __syncwarp();                                               // the stage is read
    if (lane == 0 && p + KV4_STAGES * KV4_WARPS < p1) issue(p + KV4_STAGES * KV4_WARPS, st);
  }
  if (bad) set_status(status, KID_ATTN_DECODE, FF_ERR_BOUNDS, b, split);
  if (!ok) {                                                    // a copy that never came: give those in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();                                              // the rings are free

  float* const so = reinterpret_cast<float*>(smem);             // [warp][column][D], then [warp][column][2]
  float* const sml = so + KV4_WARPS * NT * 8 * D;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = nt * 8 + 2 * t + e;
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4); l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      if (g == 0) { sml[(warp * NT * 8 + col) * 2] = m[nt][e]; sml[(warp * NT * 8 + col) * 2 + 1] = l[nt][e]; }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float add = ol[nt][j][e];
        add += __shfl_xor_sync(0xffffffffu, add, 4); add += __shfl_xor_sync(0xffffffffu, add, 8); add += __shfl_xor_sync(0xffffffffu, add, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)                             // nibble i of lane g's unit: element 32 j + 8 (g / 2) + 2 i + g % 2
          so[(warp * NT * 8 + col) * D + 32 * j + 8 * (g >> 1) + 2 * i + (g & 1)] = o[nt][j][i >> 1][2 * (i & 1) + e] + add;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < min(columns, NT * 8) * D; i += 32 * KV4_WARPS) {
    const int col = i / D, d = i - col * D;
    float M = KV4_NEG, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < KV4_WARPS; ++w) M = fmaxf(M, sml[(w * NT * 8 + col) * 2]);
#pragma unroll
    for (int w = 0; w < KV4_WARPS; ++w) {
      const float sc = exp2f(sml[(w * NT * 8 + col) * 2] - M);
      L += sml[(w * NT * 8 + col) * 2 + 1] * sc;
      acc += so[(w * NT * 8 + col) * D + d] * sc;
    }
    const int c = ct * NT * 8 + col, qi = c / G, head = kvh * G + c % G;
    if (nsplit == 1) {
      out[(size_t)(row0 + qi) * ldo + (size_t)head * D + d] = __float2bfloat16(L > 0.f ? acc / L : 0.f);
    } else {
      const size_t pr = ((size_t)(row0 + qi) * hq + head) * nsplit + split;
      part_o[pr * D + d] = acc;
      if (d == 0) part_ml[pr] = make_float2(M, L);
    }
  }
}

// Splits of one (row, head) joined; D threads each.
template <int D>
__global__ void __launch_bounds__(D)
kv4_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, __nv_bfloat16* __restrict__ out, int hq, long long ldo, int nsplit) {
  pdl_trigger();
  pdl_wait();
  const size_t pr = (size_t)blockIdx.x * nsplit;
  float M = KV4_NEG, L = 0.f, acc = 0.f;
  for (int s = 0; s < nsplit; ++s) M = fmaxf(M, part_ml[pr + s].x);
  for (int s = 0; s < nsplit; ++s) {
    const float2 v = part_ml[pr + s];
    const float sc = exp2f(v.x - M);
    L += v.y * sc;
    acc += part_o[(pr + s) * D + threadIdx.x] * sc;
  }
  const int row = blockIdx.x / hq, head = blockIdx.x - row * hq;
  out[(size_t)row * ldo + (size_t)head * D + threadIdx.x] = __float2bfloat16(L > 0.f ? acc / L : 0.f);
}

}  // namespace ff
using namespace ff;

// Splits that ff_kv4_attn_rows takes for such a launch, and the floats of scratch it needs for them (0 for one split).
FF_EXPORT int ff_kv4_attn_plan(int batch, int hq, int hkv, int nq, int dim, int max_ctx, long long* floats) {
  const int columns = nq * (hq / hkv), pages = (max_ctx + KV4_PAGE - 1) / KV4_PAGE;
  const long long ctas = (long long)batch * hkv * ((columns + 15) / 16);
  long long nsplit = (2ll * sm_count() * 2 + ctas - 1) / ctas;
  const long long most = (pages + KV4_WARPS - 1) / KV4_WARPS;
  if (nsplit > most) nsplit = most;
  if (nsplit > 128) nsplit = 128;
  if (nsplit < 1) nsplit = 1;
  if (floats) *floats = nsplit > 1 ? (long long)batch * nq * hq * nsplit * (dim + 2) : 0;
  return (int)nsplit;
}

// q rows [.., ldq] with head h at column h dim; sequence b has rows q_start[b] .. + q_lens[b], or nq rows from b nq on where those are null (only then may
// there be splits); ctx_lens[b] keys are seen by the last of them. Rows of no keys are zero.
FF_EXPORT int ff_kv4_attn_rows(const void* q, const void* kpages, const void* vpages, const int* block_table, const int* q_start, const int* q_lens,
                               const int* ctx_lens, void* out, float* scratch, int batch, int nq, int hq, int hkv, int dim, long long ldq, long long ldo,
                               int max_blocks, int num_blocks, int nsplit, float scale, int* status, cudaStream_t s) {
  if (batch <= 0 || batch > 65535 || nq <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || (dim != 64 && dim != 128) || max_blocks <= 0 || num_blocks <= 0) return FF_HOST_BAD_SHAPE;
  if (!(scale > 0.f) || nsplit < 1 || (q_start == nullptr) != (q_lens == nullptr) || (nsplit > 1 && (scratch == nullptr || q_start != nullptr))) return FF_HOST_BAD_SHAPE;
  if (ldq % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kpages) | reinterpret_cast<uintptr_t>(vpages)) & 15)) return FF_HOST_BAD_ALIGN;
  const int columns = nq * (hq / hkv);
  const bool wide = columns > 8;
  const long long tiles = (long long)hkv * (wide ? (columns + 15) / 16 : 1);
  if (tiles > 65535) return FF_HOST_TOO_LARGE;
  auto kern = dim == 128 ? (wide ? kv4_rows_kernel<128, 2> : kv4_rows_kernel<128, 1>) : (wide ? kv4_rows_kernel<64, 2> : kv4_rows_kernel<64, 1>);
  const int bytes = dim == 128 ? (wide ? kv4_smem<128, 2>() : kv4_smem<128, 1>()) : (wide ? kv4_smem<64, 2>() : kv4_smem<64, 1>());
  if (int r = opt_in_smem(kern, bytes)) return r;
  const long long rows = (long long)batch * nq;                 // with splits
  float2* ml = nsplit > 1 ? reinterpret_cast<float2*>(scratch + rows * hq * nsplit * dim) : nullptr;
  if (int r = launch_pdl(kern, dim3(nsplit, (unsigned)tiles, batch), dim3(32 * KV4_WARPS), bytes, s, 0, (const __nv_bfloat16*)q, (const uint8_t*)kpages,
                         (const uint8_t*)vpages, block_table, q_start, q_lens, ctx_lens, (__nv_bfloat16*)out, scratch, ml, nq, hq, hkv, ldq, ldo, max_blocks,
                         num_blocks, nsplit, scale * 1.4426950408889634f, status)) return r;
  if (nsplit == 1) return FF_HOST_OK;
  return launch_pdl(dim == 128 ? kv4_merge_kernel<128> : kv4_merge_kernel<64>, dim3((unsigned)(rows * hq)), dim3(dim), 0, s, 0, (const float*)scratch,
                    (const float2*)ml, (__nv_bfloat16*)out, hq, ldo, nsplit);
}
