// Prompts over the 4-bit key / value cache on the 5th-generation tensor cores (layout and format: kv4.cuh).
//
// The rows of a sequence times the query heads of one kv head are flattened (row c: query c / G, head c % G of the group), and a CTA has two tiles of 128 of
// them over one kv head: both read the same keys and values, so a page is turned into FP16 once for 256 rows. Per page j of 64 tokens:
//   one warp      fetches the page by bulk copies, three pages ahead, and finds its powers of two
//   four warps    write keys and values code * scale + lo, rounded once, as 128-byte-swizzled tiles
//   two threads   one for a tile i: S_i(j + 1) = Q_i K^T, then O_i += P_i V; S, P and O live in tensor memory (P over the S that it came from). (One thread for both
//                 spends 1400 cycles a page on issuing and on barriers, as long as the products take.)
//   two x 4 warps soft-max of a tile, a thread per row: running maximum and sum in FP32 in the base-2 domain; O is rescaled only when the maximum has moved
//                 by more than 2^8 (the stale one stays exact: P and the sum share it)
// All operands are FP16, this kernel's choice of a rounding: keys, values and weights keep 11 bits where BF16 has 8 (outputs 0.0017 off in the root mean square,
// as a single rounding of the result is; 0.0035 with BF16 operands). Whatever size they are: the warp that fetches pages finds a page's greatest |lo| and 16 scale, and its keys and
// its values are divided by a power of two of that and multiplied by 2^13 (elements stay below 2^15; what lies 2^-28 below is off by 2^-38 of the greatest). The soft-max takes the keys'
// back page by page; O is held over the values', which rises with a binade to spare and falls behind pages 2^KVT_KEPT smaller, by the path that rescales O. Weights are
// multiplied by 2^7, so that they have 11 bits down to 2^-21. Operands as they are take 584 us where this takes 599, but elements of 2^-20 were off by 8 % and more. Queries are divided by a power
// of two per row, which the soft-max's scale takes back.
// S(j + 1) of a tile waits for its P V (j - 1), whose P it overwrites; the other tile's products run meanwhile.
// 8191 rows of 32 / 8 heads of 128 from the beginning: 599 us, 918 TFLOP/s (641 in a row, at the clock that power leaves then). What the parts take was measured when operands were as they are and
// the whole took 567: the products alone 403 (S = Q K^T has 64
// columns, for which shared memory feeds the tensor cores at two thirds of their rate), the tiles of keys and values alone 475, both without the soft-max 500. They share
// shared memory (128 KB of operands a page, 42 for the tiles, some 1350 of 2050 cycles) and issue slots (54 % taken): eight warps for the tiles, with registers that the
// others give up, take 617. The warps that write the tiles wait for loads and barriers rather than for issue slots: a page read at once, one wait and one fence for
// keys and values gave 3 % back of the 6 that the powers of two took, another wait costs 7.
// Every wait is bounded; a time-out records FF_ERR_TIMEOUT, and all roles leave through the abort flag.
#include "kv4.cuh"
#include "host_util.h"

namespace ff {

constexpr int KVT_M = 128, KVT_N = KV4_PAGE, KVT_STAGES = 3;
constexpr int KVT_SOFT = 8, KVT_FILL = 4, KVT_WARPS = KVT_SOFT + KVT_FILL + 3;      // warps 0-7 soft-max, 8-11 tiles, 12 and 14 products, 13 pages
constexpr int KVT_PAGES = 3;                                                         // pages on their way or being turned into tiles (four: 627 us where three took 619)
constexpr int KVT_SIZES = 8;                                                         // pages whose sizes are known: more than are between warp 13 and the soft-max
constexpr int KVT_KEPT = 6;                                                          // binades that a page's values may lie below the power of two that they are divided by
constexpr float KVT_MOVED = 8.0f, KVT_GAIN = 7.0f;                                   // log2 units: how far a maximum may lie behind, and what weights are multiplied by
template <int D> constexpr int kvt_smem() { return 2 * KVT_M * D * 2 + 2 * KVT_STAGES * KVT_N * D * 2 + KVT_PAGES * 2 * kv4_page_bytes(D) + 1024; }

struct alignas(8) KvtBars {
  uint64_t q_full[2], k_full[KVT_STAGES], v_full[KVT_STAGES], v_empty[KVT_STAGES], s_full[2][2], p_full[2][2], pv_done[2][2], p_in[KVT_PAGES], p_out[KVT_PAGES], e_ready[KVT_SIZES];
  float2 size[KVT_SIZES];                                                              // what a page's scores are multiplied by, and O in front of it
  uint2 by[KVT_SIZES];                                                                 // its keys' and values' scale and lo, twice in BF16
  float back;                                                                          // what O is multiplied by in the end
  uint32_t tmem_base;
  int abort_flag;
};

// nibbles at bits 0 and 16 (HIGH: 4 and 20) times scale plus lo as FP16, one rounding (1024 + n, 64 + n are FP16 numbers, the difference is exact)
template <bool HIGH>
__device__ __forceinline__ uint32_t kvt_value(uint32_t w, uint32_t scale2, uint32_t lo2) {
  uint32_t n = HIGH ? (w & 0x00f000f0u) | 0x54005400u : (w & 0x000f000fu) | 0x64006400u, r;
  asm("{\n\t.reg .b32 t;\n\tadd.rn.f16x2 t, %1, %2;\n\tfma.rn.f16x2 %0, t, %3, %4;\n\t}" : "=r"(r) : "r"(n), "r"(HIGH ? 0xd400d400u : 0xe400e400u), "r"(scale2), "r"(lo2));
  return r;
}

template <int D>
__device__ __forceinline__ void kvt_load(uint32_t (&dst)[D / 32], uint32_t src) {
  if (D == 128) kv4_lds(src, dst[0], dst[1], dst[D / 32 - 2], dst[D / 32 - 1]);
  else kv4_lds(src, dst[0], dst[1]);
}

// Several sequences of long contexts, which differ: one CTA makes a list of what there is to do, long tile pairs cut into pieces of equal size, the largest first (the
// next SM that is free takes the next one). Each is a CTA of the kernel below for every kv head. Two tile pairs of 470 pages beside sixty of 90 and less: 530 us as they
// lie, 365 so.
struct KvtPlan {
  int* count;             // pieces; tile pairs of more than one
  int4* item;             // piece: sequence, first flattened row, first page, pages
  int4* join;             // tile pair of more than one: sequence, first flattened row, pieces, slot of the first
  int* slot;              // where a piece leaves its part of the result, -1: it is the only one
  int items, joins, slots;
};
// A piece is at most as large as the longest tile pair, or as an SM's share of all pages over 1, 1.5 or 2 (KVT_SHARE): whichever should end first.
constexpr int KVT_PLAN_WARPS = 16, KVT_CLASSES = 32, KVT_CUTS = 4, KVT_SHARE = 2;
constexpr int KVT_EXTRA = 6, KVT_PART = 4;                                // pages' time that a CTA takes beside its pages, and for a part's way out and in again
constexpr int KVT_SEQS = 2048;                                            // sequences of a list at most
// Pages of a context from which a list is made. It takes 6 us and more where it cuts: 100 x 5 rows behind up to 2000 tokens 80 us as they lie and 93 by a list, 8 x 64 behind up to 4000 67 and 63, 500
// of 4 behind 60000 374 and 116. It is not right for every call: 4 x 5 rows (64 / 4 heads) behind up to 30000 take 73 and 83, 10 x 16 behind 10000 124 and 132, 24 x 5 behind up to 4000 61 and 65.
constexpr int KVT_LIST = 32;

__device__ __forceinline__ int kvt_pages(int past, int c0, int rows, int G) { return (max(past + (c0 + min(rows, 2 * KVT_M) - 1) / G + 1, 0) + KVT_N - 1) / KVT_N; }

__global__ void __launch_bounds__(32 * KVT_PLAN_WARPS)
kv4_plan_kernel(const KvtPlan plan, const int* __restrict__ q_start, const int* __restrict__ q_lens, const int* __restrict__ ctx_lens, int batch, int all_rows, int nq, int G,
                int hkv, int max_blocks, int sms, int* status) {
  __shared__ int s_n[KVT_SEQS], s_past[KVT_SEQS];
  __shared__ unsigned long long s_all;
  __shared__ int s_most, s_class[KVT_CUTS][KVT_CLASSES], s_slots, s_joins;
  __shared__ float s_end[KVT_CUTS];
  __shared__ int s_pieces[KVT_CUTS];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < KVT_CUTS * KVT_CLASSES) s_class[threadIdx.x / KVT_CLASSES][threadIdx.x % KVT_CLASSES] = 0;
  if (threadIdx.x == 0) { s_all = 0; s_most = 1; s_slots = 0; s_joins = 0; }
  pdl_wait();
  for (int b = threadIdx.x; b < batch; b += 32 * KVT_PLAN_WARPS) {
    int n = q_lens ? q_lens[b] : nq;
    const int row0 = q_start ? q_start[b] : b * nq, ctx = ctx_lens[b];
    if (n > 0 && (n > nq || row0 < 0 || n > all_rows - row0)) {   // rows that the call does not have
      set_status(status, KID_ATTN_PREFILL, FF_ERR_BOUNDS, b, row0);
      n = 0;
    }
    s_n[b] = max(n, 0);
    s_past[b] = min(max(ctx, 0), max_blocks * KV4_PAGE) - n;
  }
  __syncthreads();
  auto each = [&](auto&& f) {                                    // f(sequence, first row, pages) for every tile pair: a warp has a sequence, a lane a tile pair
    for (int b = warp; b < batch; b += KVT_PLAN_WARPS) {
      const int n = s_n[b], past = s_past[b];
      for (int c0 = lane * 2 * KVT_M; c0 < n * G; c0 += 32 * 2 * KVT_M) f(b, c0, kvt_pages(past, c0, n * G - c0, G));
    }
  };
  unsigned long long all = 0;
  int most = 1;
  each([&](int, int, int pages) { all += pages + KVT_EXTRA; most = max(most, pages); });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { all += __shfl_xor_sync(0xffffffffu, all, o); most = max(most, __shfl_xor_sync(0xffffffffu, most, o)); }
  if (lane == 0) { atomicAdd(&s_all, all); atomicMax(&s_most, most); }
  __syncthreads();
  most = s_most;
  // sizes to choose from (at most 128 pieces of a tile pair), and how many pieces of which size each gives (size classes, the largest first)
  const float share = (float)s_all * hkv / sms;
  auto size_of = [&](int j) { return j == 0 ? most : min(most, max((int)min(share / (0.5f + 0.5f * j) + 1.f, 1.0e9f), max(4, (most + 127) / 128))); };
  auto cut = [&](int pages, int size, int& ns, int& per) { ns = max((pages + size - 1) / size, 1); per = (pages + ns - 1) / ns; };
  auto size_class = [&](int per) { return KVT_CLASSES - 1 - (int)((long long)per * (KVT_CLASSES - 1) / most); };
  int sizes[KVT_CUTS];
#pragma unroll
  for (int j = 0; j < KVT_CUTS; ++j) sizes[j] = size_of(j);
  each([&](int, int, int pages) {
#pragma unroll
    for (int j = 0; j < KVT_CUTS; ++j) { int ns, per; cut(pages, sizes[j], ns, per); atomicAdd(&s_class[j][size_class(per)], ns); }
  });
  __syncthreads();
  if (warp < KVT_CUTS) {
    // When the last piece should end: not before an SM's share of them all, nor before i + 1 times the (i sms + 1)-th largest, as one SM has i + 1 of these
    const int own = s_class[warp][lane];
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
    const float pages = (float)(KVT_CLASSES - 1 - lane) * most / (KVT_CLASSES - 1) + KVT_EXTRA + (warp > 0 ? KVT_PART : 0);
    float end = own > 0 ? (float)(((long long)sum * hkv - 1) / sms + 1) * pages : 0.f, work = own * pages;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { end = fmaxf(end, __shfl_xor_sync(0xffffffffu, end, o)); work += __shfl_xor_sync(0xffffffffu, work, o); }
    if (lane == 0) s_end[warp] = fmaxf(end, work * hkv / sms);
    __syncwarp();
    s_class[warp][lane] = sum - own;
    if (lane == 31) s_pieces[warp] = sum;
  }
  __syncthreads();
  int best = 0;
#pragma unroll
  for (int j = 1; j < KVT_CUTS; ++j)
    if (s_end[j] < s_end[best] * 0.97f) best = j;
  const int size = size_of(best);
  if (threadIdx.x == 0) plan.count[0] = min(s_pieces[best], plan.items);
  each([&](int b, int c0, int pages) {
    int ns, per;
    cut(pages, size, ns, per);
    const int at = atomicAdd(&s_class[best][size_class(per)], ns);
    int slot = -1, j = 0;
    if (ns > 1) {
      slot = atomicAdd(&s_slots, ns);
      j = atomicAdd(&s_joins, 1);
    }
    if (at + ns > plan.items || (ns > 1 && (slot + ns > plan.slots || j >= plan.joins))) {      // (sequences that overlap have more rows than there is room for)
      set_status(status, KID_ATTN_PREFILL, FF_ERR_BOUNDS, b, c0);
      for (int s = at; s < min(at + ns, plan.items); ++s) { plan.item[s] = make_int4(-1, 0, 0, 0); plan.slot[s] = -1; }
      if (ns > 1 && j < plan.joins) plan.join[j] = make_int4(b, c0, 0, 0);
      return;
    }
    for (int s = 0; s < ns; ++s) {
      plan.item[at + s] = make_int4(b, c0, s * per, max(0, min(pages - s * per, per)));
      plan.slot[at + s] = ns > 1 ? slot + s : -1;
    }
    if (ns > 1) plan.join[j] = make_int4(b, c0, ns, slot);
  });
  __syncthreads();
  if (threadIdx.x == 0) plan.count[1] = min(s_joins, plan.joins);
}

template <int D>
__global__ void __launch_bounds__(32 * KVT_WARPS, 1)
kv4_tiles_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ kpages, const uint8_t* __restrict__ vpages, const int* __restrict__ block_table,
                 const int* __restrict__ q_start, const int* __restrict__ q_lens, const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out,
                 float* __restrict__ part_o, float2* __restrict__ part_ml, const KvtPlan plan, int all_rows, int nq, int hq, int hkv, long long ldq, long long ldo, int max_blocks, int num_blocks, int nsplit,
                 float scale_log2, int* status) {
  constexpr int NG = D / 32, PB = kv4_page_bytes(D), TILE = KVT_N * D * 2, QTILE = KVT_M * D * 2;
  pdl_trigger();
  pdl_wait();
  const int G = hq / hkv;
  int b = blockIdx.z, kvh = blockIdx.y, c0 = 0, first = 0, tiles = 0, slot = -1;
  if (plan.count != nullptr) {
    const int at = blockIdx.x / hkv;
    kvh = blockIdx.x - at * hkv;
    if (at >= plan.count[0]) return;
    const int4 v = plan.item[at];
    b = v.x; c0 = v.y; first = v.z; tiles = v.w;
    slot = plan.slot[at];
    if (b < 0) return;
  } else {
    c0 = (int)((gridDim.x - 1 - blockIdx.x) / nsplit) * 2 * KVT_M;        // late rows see the most keys: they start first
  }
  const int n = q_lens ? q_lens[b] : nq;
  const int row0 = q_start ? q_start[b] : b * nq;
  if (n > 0 && (n > nq || row0 < 0 || n > all_rows - row0)) {             // rows that the call does not have
    if (threadIdx.x == 0) set_status(status, KID_ATTN_PREFILL, FF_ERR_BOUNDS, b, row0);
    return;
  }
  const int rows = n * G - c0;                                            // of this CTA and behind it
  if (rows <= 0) return;
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvtBars bars;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const sQ = smem;
  uint8_t* const sK = smem + 2 * QTILE;
  uint8_t* const sV = sK + KVT_STAGES * TILE;
  uint8_t* const sP = sV + KVT_STAGES * TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int two = rows > KVT_M ? 2 : 1;                                   // tiles of this CTA
  int ctx = max(ctx_lens[b], 0);
  if (ctx > max_blocks * KV4_PAGE) {
    if (threadIdx.x == 0) set_status(status, KID_ATTN_PREFILL, FF_ERR_BOUNDS, b, ctx);
    ctx = max_blocks * KV4_PAGE;
  }
  const int past = ctx - n;
  if (plan.count == nullptr) {
    const int pages = kvt_pages(past, c0, rows, G), per = max((pages + nsplit - 1) / nsplit, 4), split = blockIdx.x % nsplit;
    first = split * per;
    tiles = max(0, min(pages, first + per) - first);
    if (nsplit > 1) slot = (int)(b * (gridDim.x / nsplit) + c0 / (2 * KVT_M)) * nsplit + split;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_full[i], 4);
      for (int k = 0; k < 2; ++k) { mbar_init(&bars.s_full[i][k], 1); mbar_init(&bars.p_full[i][k], 4); mbar_init(&bars.pv_done[i][k], 1); }
    }
    for (int i = 0; i < KVT_STAGES; ++i) {
      mbar_init(&bars.k_full[i], KVT_FILL); mbar_init(&bars.v_full[i], KVT_FILL); mbar_init(&bars.v_empty[i], two);
    }
    for (int i = 0; i < KVT_PAGES; ++i) { mbar_init(&bars.p_in[i], 1); mbar_init(&bars.p_out[i], KVT_FILL); }
    for (int i = 0; i < KVT_SIZES; ++i) mbar_init(&bars.e_ready[i], 1);
    bars.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == KVT_SOFT + KVT_FILL) { tmem_alloc(&bars.tmem_base, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // S buffer k of tile i: columns 128 i + 64 k, its P over the first 32 of them; O of tile i: columns 256 + 128 i
  const uint32_t tmem = bars.tmem_base;
  volatile int* const abort_flag = &bars.abort_flag;

  if (warp >= KVT_SOFT && warp < KVT_SOFT + KVT_FILL) {
    // ================================ tiles of keys and values ================================
    // tokens key and key + 32, chunk u of each of their groups: the eight lanes of a store have eight tokens, whose swizzled chunks lie in different banks
    const int key0 = (warp - KVT_SOFT) * 8 + (lane & 7), u = lane >> 3;
    RingPos pr, tr;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      if (!mbar_wait(&bars.e_ready[j % KVT_SIZES], (j / KVT_SIZES) & 1, abort_flag, status, KID_ATTN_PREFILL, 40)) ok = false;
      // (its values multiplied, the keys of a stage are too)
      if (!mbar_wait(&bars.v_empty[tr.s], tr.ph ^ 1, abort_flag, status, KID_ATTN_PREFILL, 41)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint32_t page = smem_u32(sP) + pr.s * 2 * PB;
      const uint2 by = bars.by[j % KVT_SIZES];
      uint32_t code[2][2][NG], stat[2][2][NG];
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = key0 + 32 * i;
          kvt_load<D>(code[part][i], page + part * PB + (part ? kv4_value_at<D>(key, 2 * u, 0) : key * (D / 2) + u * (D / 8)));
          kvt_load<D>(stat[part][i], page + part * PB + kv4_code_bytes(D) + key * (D / 8));
        }
      if ((first + j) * KVT_N + KVT_N > ctx) {                   // behind the sequence
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if ((first + j) * KVT_N + key0 + 32 * i >= ctx) stat[0][i][g] = stat[1][i][g] = 0u;
      }
#pragma unroll
      for (int part = 0; part < 2; ++part) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t v[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 sl = unpack_bf16x2(kv4_mul2(stat[part][i][g], part ? by.y : by.x));
            const uint32_t scale2 = kv4_f16x2(sl.x, sl.x), lo2 = kv4_f16x2(sl.y, sl.y);
            // values: 16-bit unit g of two chunks, the even elements and the odd ones
            const uint32_t word = part ? kv4_prmt(code[1][i][g / 2], code[1][i][NG / 2 + g / 2], (g & 1) ? 0x7632u : 0x5410u) : code[0][i][g];
            v[i][0] = kvt_value<false>(word, scale2, lo2); v[i][1] = kvt_value<true>(word, scale2, lo2);
            v[i][2] = kvt_value<false>(word >> 8, scale2, lo2); v[i][3] = kvt_value<true>(word >> 8, scale2, lo2);
          }
          const int c = 4 * g + u;                               // 16-byte chunk of the row: 64-element block c / 8
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = key0 + 32 * i;
            kv4_sts(smem_u32(part ? sV : sK) + tr.s * TILE + key * 128 + (c >> 3) * (KVT_N * 128) + (((c & 7) ^ (key & 7)) << 4), v[i][0], v[i][1], v[i][2], v[i][3]);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) { mbar_arrive(&bars.k_full[tr.s]); mbar_arrive(&bars.v_full[tr.s]); mbar_arrive(&bars.p_out[pr.s]); }
      pr.next(KVT_PAGES);
      tr.next(KVT_STAGES);
    }
  } else if (warp == KVT_SOFT + KVT_FILL + 1) {
    // ================================ pages ================================
    // A page is fetched, and the one before it gets its powers of two: 2^13 over the one that the greatest of |lo| and 16 scale lies in, so that elements are below 2^15
    bool bad = false;
    RingPos pr, sr;
    int ref = 0, top = 0;
    int blk = tiles > 0 ? block_table[(size_t)b * max_blocks + first] : 0;
    for (int i = 0; i <= tiles && tiles > 0; ++i) {
      if (i < tiles) {
        const int next = i + 1 < tiles ? block_table[(size_t)b * max_blocks + first + i + 1] : 0;
        if (blk < 0 || blk >= num_blocks) { bad = true; blk = 0; }
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.p_out[pr.s], pr.ph ^ 1, abort_flag, status, KID_ATTN_PREFILL, 39))) break;
        if (lane == 0) {
          const size_t at = ((size_t)blk * hkv + kvh) * PB;
          mbar_expect_tx(&bars.p_in[pr.s], 2 * PB);
          kv4_bulk_load(sP + pr.s * 2 * PB, kpages + at, PB, &bars.p_in[pr.s]);
          kv4_bulk_load(sP + pr.s * 2 * PB + PB, vpages + at, PB, &bars.p_in[pr.s]);
        }
        __syncwarp();
        pr.next(KVT_PAGES);
        blk = next;
      }
      if (i == 0) continue;
      const int j = i - 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.p_in[sr.s], sr.ph, abort_flag, status, KID_ATTN_PREFILL, 38))) break;
      int ex[2];
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint32_t at = smem_u32(sP) + sr.s * 2 * PB + part * PB + kv4_code_bytes(D) + 16 * lane;
        uint32_t st[NG / 2][4], most = 0u;
#pragma unroll
        for (int h = 0; h < NG / 2; ++h) kv4_lds(at + 512 * h, st[h][0], st[h][1], st[h][2], st[h][3]);
        if ((first + j) * KVT_N + KVT_N > ctx) {                 // behind the sequence: whatever the page holds there is no number
#pragma unroll
          for (int h = 0; h < NG / 2; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((first + j) * KVT_N + (4 * (lane + 32 * h) + k) / NG >= ctx) st[h][k] = 0u;
        }
#pragma unroll
        for (int h = 0; h < NG / 2; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k) most = kv4_maxabs2(most, st[h][k]);
        ex[part] = max((int)(kv4_warp_max(max((most & 0x7fffu) + 0x0200u, most >> 16 & 0x7fffu)) >> 7), KV4_LEAST);
      }
      // O is held over the values' power: it rises with a binade to spare, and falls only behind much smaller pages
      const int before = j > 0 ? ref : ex[1] + 1;
      if (ex[1] > ref) ref = ex[1] + 1;
      else if (ex[1] + KVT_KEPT < ref) ref = max(ex[1] + 1, top - KV4_SPAN);
      top = max(top, ref);
      if (lane == 0) {
        bars.size[j % KVT_SIZES] = make_float2(__uint_as_float((uint32_t)(ex[0] - 13) << 23), __uint_as_float((uint32_t)(127 + before - ref) << 23));
        bars.by[j % KVT_SIZES] = make_uint2((uint32_t)(267 - ex[0]) * 0x00800080u, (uint32_t)(267 - ref) * 0x00800080u);
        if (j == tiles - 1) bars.back = __uint_as_float((uint32_t)(ref - 13) << 23);
        mbar_arrive(&bars.e_ready[j % KVT_SIZES]);
      }
      sr.next(KVT_PAGES);
    }
    if (bad && lane == 0) set_status(status, KID_ATTN_PREFILL, FF_ERR_BOUNDS, b, c0);
  } else if (warp >= KVT_SOFT + KVT_FILL) {
    // ================================ products: a warp for each tile ================================
    const int i = warp == KVT_SOFT + KVT_FILL ? 0 : 1;
    if (i < two && tiles > 0 && elect_one()) {
      const uint32_t idesc_s = umma_idesc(0, 0, 0, 0, KVT_M, KVT_N), idesc_o = umma_idesc(0, 0, 0, 1, KVT_M, D);
      // descriptors differ by byte offsets / 16 in their low bits
      const uint64_t qd = umma_desc_sw128(smem_u32(sQ) + i * QTILE, 16, 1024), kd = umma_desc_sw128(smem_u32(sK), 16, 1024), vd = umma_desc_sw128(smem_u32(sV), KVT_N * 128, 1024);
      const uint32_t s_at = tmem + 128 * i, o_at = tmem + 256 + 128 * i;
      bool ok = mbar_wait(&bars.q_full[i], 0, abort_flag, status, KID_ATTN_PREFILL, 43);
      RingPos kr, vr;
      auto issue_s = [&](int j) -> bool {
        if (!mbar_wait(&bars.k_full[kr.s], kr.ph, abort_flag, status, KID_ATTN_PREFILL, 44)) return false;
        // the buffer holds the P of page j - 2
        if (j >= 2 && !mbar_wait(&bars.pv_done[i][j & 1], ((j >> 1) & 1) ^ 1, abort_flag, status, KID_ATTN_PREFILL, 50)) return false;
        tc_fence_after();
        const uint64_t d = kd + (uint32_t)(kr.s * (TILE >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(s_at + 64 * (j & 1), qd + (uint32_t)(((k >> 2) * (KVT_M * 128) + (k & 3) * 32) >> 4), d + (uint32_t)(((k >> 2) * (KVT_N * 128) + (k & 3) * 32) >> 4), idesc_s, k != 0);
        umma_commit(&bars.s_full[i][j & 1]);
        kr.next(KVT_STAGES);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; j < tiles && ok; ++j) {
        if (j + 1 < tiles && !issue_s(j + 1)) { ok = false; break; }
        if (!mbar_wait(&bars.v_full[vr.s], vr.ph, abort_flag, status, KID_ATTN_PREFILL, 45)) { ok = false; break; }
        if (!mbar_wait(&bars.p_full[i][j & 1], (j >> 1) & 1, abort_flag, status, KID_ATTN_PREFILL, 46)) { ok = false; break; }
        tc_fence_after();
        const uint64_t d = vd + (uint32_t)(vr.s * (TILE >> 4));
#pragma unroll
        for (int k = 0; k < KVT_N / 16; ++k)
          umma_f16_ts(o_at, s_at + 64 * (j & 1) + k * 8, d + (uint32_t)((k * 2048) >> 4), idesc_o, (j > 0) || (k != 0));
        umma_commit(&bars.pv_done[i][j & 1]);
        umma_commit(&bars.v_empty[vr.s]);
        vr.next(KVT_STAGES);
      }
    }
  } else {
    // ================================ soft-max ================================
    const int i = warp >> 2, row = (warp & 3) * 32 + lane;               // tile, row = lane of tensor memory
    if (i < two) {
      const int c = c0 + i * KVT_M + row;
      const bool live = c < n * G;
      const int qi = live ? c / G : 0, head = kvh * G + (live ? c - qi * G : 0);
      float row_scale = scale_log2;
      {
        // The row as FP16, divided by the power of two of its greatest element: exact, but for elements below 2^-14 of that.
        uint32_t w[D / 2];
        const uint4* src = reinterpret_cast<const uint4*>(q + (size_t)(row0 + qi) * ldq + (size_t)head * D);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          const uint4 v = live ? src[k] : make_uint4(0, 0, 0, 0);
          w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
        }
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < D / 2; ++k) { const float2 v = unpack_bf16x2(w[k]); most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y))); }
        const uint32_t e = min(max(__float_as_uint(most) >> 23, 2u), 252u);          // 2^(e - 127), and its inverse
        const float up = __uint_as_float(e << 23), down = __uint_as_float((254u - e) << 23);
        row_scale *= up;
        const uint32_t dst = smem_u32(sQ) + i * QTILE + row * 128;
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          uint32_t x[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) { const float2 v = unpack_bf16x2(w[4 * k + z]); x[z] = kv4_f16x2(v.x * down, v.y * down); }
          kv4_sts(dst + (k >> 3) * (KVT_M * 128) + (((k & 7) ^ (row & 7)) << 4), x[0], x[1], x[2], x[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[i]);
      }
      const int hi = live ? past + qi : -1;
      const int all = past + (c0 + i * KVT_M) / G;                       // keys up to here are seen by every row of the tile
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tmem_o = tmem + 256 + 128 * i + lanes;
      float m_ref = -INFINITY;
      float l0 = 0.f, l1 = 0.f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        const uint32_t s_addr = tmem + 128 * i + 64 * (j & 1) + lanes;
        {
          const bool sized = mbar_try_wait(&bars.e_ready[j % KVT_SIZES], (j / KVT_SIZES) & 1), there = mbar_try_wait(&bars.s_full[i][j & 1], (j >> 1) & 1);
          if (!sized && !mbar_wait(&bars.e_ready[j % KVT_SIZES], (j / KVT_SIZES) & 1, abort_flag, status, KID_ATTN_PREFILL, 51)) ok = false;
          if (!there && !mbar_wait(&bars.s_full[i][j & 1], (j >> 1) & 1, abort_flag, status, KID_ATTN_PREFILL, 47)) ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const float2 size = bars.size[j % KVT_SIZES];
        const float page_scale = fmaxf(row_scale * size.x, 1.1754944e-38f);      // (times minus infinity it has to be that)
        float s[KVT_N];
        {
          uint32_t r[KVT_N];
          tmem_ld_x32(s_addr, r);
          tmem_ld_x32(s_addr + 32, r + 32);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < KVT_N; ++k) s[k] = __uint_as_float(r[k]);
        }
        if ((first + j) * KVT_N + KVT_N - 1 > all) {
#pragma unroll
          for (int k = 0; k < KVT_N; ++k) s[k] = (first + j) * KVT_N + k <= hi ? s[k] : -INFINITY;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < KVT_N; ++k) mx4[k & 3] = fmaxf(mx4[k & 3], s[k]);
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * page_scale;
        float alpha = 1.f;
        bool need = false;
        if (mx > m_ref + KVT_MOVED || (m_ref == -INFINITY && mx > -INFINITY)) {
          alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
          m_ref = mx;
          need = j > 0;
        }
        need = need || size.y != 1.f;                                    // (1 for the first page)
        if (__any_sync(0xffffffffu, need)) {
          // O is rescaled in place: the P V before has to be complete (the rare path)
          if (!mbar_wait(&bars.pv_done[i][(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, status, KID_ATTN_PREFILL, 48)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const float by = alpha * size.y;
#pragma unroll
          for (int k = 0; k < D; k += 16) {
            uint32_t r[16];
            tmem_ld_x16(tmem_o + k, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * by);
            tmem_st_x16(tmem_o + k, r);
          }
          tmem_st_wait();
        }
        const float mr = m_ref == -INFINITY ? 0.f : m_ref;
        const uint64_t scale2 = f2_pack(page_scale, page_scale), off2 = f2_pack(KVT_GAIN - mr, KVT_GAIN - mr);
        uint64_t sum = f2_pack(l0 * alpha, l1 * alpha);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float a, e;
            f2_unpack(f2_fma(f2_pack(s[32 * h + 2 * k], s[32 * h + 2 * k + 1]), scale2, off2), a, e);
            a = kv4_ex2(a); e = kv4_ex2(e);
            pk[k] = kv4_f16x2(a, e);
            sum = f2_add(sum, f2_pack(a, e));
          }
          tmem_st_x16(s_addr + 16 * h, pk);
        }
        f2_unpack(sum, l0, l1);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[i][j & 1]);
      }
      if (ok && tiles > 0 && !mbar_wait(&bars.pv_done[i][(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, abort_flag, status, KID_ATTN_PREFILL, 49)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        const float l = l0 + l1, inv = l == 0.f ? 0.f : 1.f / l, back = tiles > 0 ? bars.back : 1.f;
        __nv_bfloat16* dst = out + (size_t)(row0 + qi) * ldo + (size_t)head * D;
        const size_t pr = ((size_t)slot * hkv + kvh) * (2 * KVT_M) + i * KVT_M + row;
        if (slot >= 0 && live) part_ml[pr] = make_float2(m_ref == -INFINITY ? -3.0e38f : m_ref, l);
#pragma unroll
        for (int k = 0; k < D; k += 16) {
          uint32_t r[16];
          if (tiles > 0) { tmem_ld_x16(tmem_o + k, r); tmem_ld_wait(); }
          if (!live) continue;
          if (slot >= 0) {
            if (l != 0.f) {                                      // (the merge does not read what has no weight)
#pragma unroll
              for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(part_o + pr * D + k + e) =
                  make_float4(__uint_as_float(r[e]) * back, __uint_as_float(r[e + 1]) * back, __uint_as_float(r[e + 2]) * back, __uint_as_float(r[e + 3]) * back);
            }
            continue;
          }
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = l == 0.f ? 0u : pack_bf16x2(__uint_as_float(r[2 * e]) * inv * back, __uint_as_float(r[2 * e + 1]) * inv * back);
          reinterpret_cast<uint4*>(dst + k)[0] = make_uint4(o[0], o[1], o[2], o[3]);
          reinterpret_cast<uint4*>(dst + k)[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (bars.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (warp == KVT_SOFT + KVT_FILL) { __syncwarp(); tc_fence_after(); tmem_dealloc(bars.tmem_base, 512); }
}

// The pieces of a tile pair joined: a warp per row, a lane D / 32 elements, four pieces on their way at once.
constexpr int KVT_JOIN = 8;                                               // rows of a CTA
template <int D>
__global__ void __launch_bounds__(256)
kv4_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const KvtPlan plan, const int* __restrict__ q_start, const int* __restrict__ q_lens,
                __nv_bfloat16* __restrict__ out, int batch, int tiles, int all_rows, int nq, int hq, int hkv, long long ldo, int nsplit) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = hq / hkv, count = plan.count != nullptr ? plan.count[1] : tiles * batch;
  const int chunks = (min(nq * G, 2 * KVT_M) + KVT_JOIN - 1) / KVT_JOIN;                                          // of a tile pair
  for (long long w = blockIdx.x; w < (long long)count * hkv * chunks; w += gridDim.x) {
    const int th = (int)(w / chunks), t = th / hkv, kvh = th - t * hkv, r0 = (int)(w - (long long)th * chunks) * KVT_JOIN;
    const int4 v = plan.count != nullptr ? plan.join[t] : make_int4(t / tiles, t % tiles * 2 * KVT_M, nsplit, t * nsplit);
    const int b = v.x, c0 = v.y, ns = v.z, n = q_lens ? q_lens[b] : nq, row0 = q_start ? q_start[b] : b * nq;
    if (n > nq || row0 < 0 || n > all_rows - row0) continue;
    for (int r = r0 + warp; r < min(r0 + KVT_JOIN, n * G - c0); r += 8) {
      const int qi = (c0 + r) / G, head = kvh * G + c0 + r - qi * G;
      const size_t first = ((size_t)v.w * hkv + kvh) * (2 * KVT_M) + r, step = (size_t)hkv * (2 * KVT_M);
      float2 ml[4];                                                         // of pieces lane, lane + 32, ... (at most 128)
      float M = -3.0e38f, L = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i] = lane + 32 * i < ns ? part_ml[first + (lane + 32 * i) * step] : make_float2(-3.0e38f, 0.f);
        M = fmaxf(M, ml[i].x);
      }
      M = warp_max(M);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i].x = ml[i].y == 0.f ? 0.f : kv4_ex2(ml[i].x - M);              // (a piece of no weight has left nothing)
        L = fmaf(ml[i].y, ml[i].x, L);
      }
      L = warp_sum(L);
      float acc[E];
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int s = 32 * i; s < min(ns, 32 * i + 32); s += 4) {
          float v4[4][E], sc[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            sc[u] = __shfl_sync(0xffffffffu, ml[i].x, (s + u) & 31);        // (0 behind the last piece)
#pragma unroll
            for (int k = 0; k < E; ++k) v4[u][k] = 0.f;
            if (sc[u] != 0.f) {
              const float* src = part_o + (first + (s + u) * step) * D + lane * E;
              if constexpr (E == 4) { const float4 x = *reinterpret_cast<const float4*>(src); v4[u][0] = x.x; v4[u][1] = x.y; v4[u][2] = x.z; v4[u][3] = x.w; }
              else { const float2 x = *reinterpret_cast<const float2*>(src); v4[u][0] = x.x; v4[u][1] = x.y; }
            }
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] = fmaf(v4[u][k], sc[u], acc[k]);
        }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      uint32_t* dst = reinterpret_cast<uint32_t*>(out + (size_t)(row0 + qi) * ldo + (size_t)head * D) + lane * (E / 2);
#pragma unroll
      for (int k = 0; k < E / 2; ++k) dst[k] = pack_bf16x2(acc[2 * k] * inv, acc[2 * k + 1] * inv);
    }
  }
}

// What a call's scratch has room for. List (nsplit 0): pieces are KVT_SHARE times the SMs at most and one for every tile pair; a tile pair that is cut has no more than
// twice as many as it is sizes large.
struct KvtRoom { long long each, tiles, items, joins, slots, ints; };        // each: tile pairs of a sequence at most, tiles: of all
static KvtRoom kvt_room(int batch, int rows, int max_q_len, int hq, int hkv, int nsplit) {
  const long long G = hq / hkv, each = ((long long)(max_q_len < rows ? max_q_len : rows) * G + 2 * KVT_M - 1) / (2 * KVT_M), some = ((long long)rows * G + 2 * KVT_M - 1) / (2 * KVT_M);
  KvtRoom r{};
  r.each = each;
  r.tiles = batch * each < batch + some ? batch * each : batch + some;
  if (nsplit == 0) {
    r.joins = KVT_SHARE * sm_count() / hkv + 1;
    r.items = r.tiles + r.joins;
    r.slots = 2 * r.joins;
    r.ints = (4 + 5 * r.items + 4 * r.joins + 3) / 4 * 4;
  } else if (nsplit > 1) {
    r.slots = batch * each * nsplit;
  }
  return r;
}

}  // namespace ff
using namespace ff;

// Splits of ff_kv4_attn_tiles (0: by a list), and the floats of scratch it needs. rows: of the whole call, at most max_q_len per sequence. One CTA stands on an SM. One
// sequence, or contexts of few pages: where there are fewer CTAs than SMs the keys are split, down to four pages each: for one round of CTAs, or three where more than
// half of the SMs have one (96 CTAs of up to 62 pages 66 us, in three splits 61). That counts as many tile pairs for every sequence as the longest has, which is also what
// their parts' room is made for.
FF_EXPORT int ff_kv4_tiles_plan(int batch, int rows, int max_q_len, int hq, int hkv, int dim, int max_ctx, long long* floats) {
  const long long ctas = kvt_room(batch, rows, max_q_len, hq, hkv, 1).each * hkv * batch, most = (max_ctx + 4 * KVT_N - 1) / (4 * KVT_N);
  long long nsplit = ctas <= 0 ? 1 : 2 * ctas <= sm_count() ? sm_count() / ctas : ctas < sm_count() ? 3 : 1;
  if (nsplit > most) nsplit = most;
  if (nsplit > 128) nsplit = 128;
  if (nsplit < 1) nsplit = 1;
  if (batch > 1 && batch <= KVT_SEQS && max_ctx >= KVT_LIST * KVT_N) nsplit = 0;
  const KvtRoom r = kvt_room(batch, rows, max_q_len, hq, hkv, (int)nsplit);
  if (floats) *floats = r.ints + r.slots * hkv * 2 * KVT_M * (dim + 2);
  return (int)nsplit;
}

// As ff_kv4_attn_rows; out rows of whole 16 bytes. rows: of q and out.
FF_EXPORT int ff_kv4_attn_tiles(const void* q, const void* kpages, const void* vpages, const int* block_table, const int* q_start, const int* q_lens,
                                const int* ctx_lens, void* out, float* scratch, int batch, int rows, int max_q_len, int hq, int hkv, int dim, long long ldq, long long ldo,
                                int max_blocks, int num_blocks, int nsplit, float scale, int* status, cudaStream_t s) {
  if (batch <= 0 || batch > 65535 || rows <= 0 || max_q_len <= 0 || hq <= 0 || hkv <= 0 || hkv > 65535 || hq % hkv || (dim != 64 && dim != 128) || max_blocks <= 0 || num_blocks <= 0)
    return FF_HOST_BAD_SHAPE;
  if (q_start == nullptr && (long long)batch * max_q_len != rows) return FF_HOST_BAD_SHAPE;
  if (!(scale > 0.f) || (q_start == nullptr) != (q_lens == nullptr) || !ctx_lens || nsplit < 0 || nsplit > 128 || (nsplit == 0 && batch > KVT_SEQS) || (nsplit != 1 && scratch == nullptr)) return FF_HOST_BAD_SHAPE;
  if (ldq % 8 || ldo % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kpages) | reinterpret_cast<uintptr_t>(vpages) | reinterpret_cast<uintptr_t>(out) |
                              reinterpret_cast<uintptr_t>(scratch)) & 15))
    return FF_HOST_BAD_ALIGN;
  const KvtRoom room = kvt_room(batch, rows, max_q_len, hq, hkv, nsplit);
  if (max_q_len > rows) max_q_len = rows;
  const long long columns = (long long)max_q_len * (hq / hkv), each = room.each, grid = nsplit ? each * nsplit : room.items * hkv;
  if (columns > 0x7fffff00ll || grid > 0x7fffffffll || room.slots > 0x7fffffffll) return FF_HOST_TOO_LARGE;
  auto kern = dim == 128 ? kv4_tiles_kernel<128> : kv4_tiles_kernel<64>;
  const int bytes = dim == 128 ? kvt_smem<128>() : kvt_smem<64>();
  if (int r = opt_in_smem(kern, bytes)) return r;
  float* const part = scratch + room.ints;
  float2* const ml = reinterpret_cast<float2*>(part + room.slots * hkv * 2 * KVT_M * dim);
  KvtPlan plan{};
  if (nsplit == 0) {
    int* at = reinterpret_cast<int*>(scratch);
    plan.count = at; at += 4;
    plan.item = reinterpret_cast<int4*>(at); at += 4 * room.items;
    plan.join = reinterpret_cast<int4*>(at); at += 4 * room.joins;
    plan.slot = at;
    plan.items = (int)room.items; plan.joins = (int)room.joins; plan.slots = (int)room.slots;
    if (int r = launch_pdl(kv4_plan_kernel, dim3(1), dim3(32 * KVT_PLAN_WARPS), 0, s, 0, plan, q_start, q_lens, ctx_lens, batch, rows, max_q_len, hq / hkv, hkv, max_blocks,
                           sm_count(), status)) return r;
  }
  if (int r = launch_pdl(kern, nsplit ? dim3((unsigned)grid, hkv, batch) : dim3((unsigned)grid), dim3(32 * KVT_WARPS), bytes, s, 0, (const __nv_bfloat16*)q, (const uint8_t*)kpages,
                         (const uint8_t*)vpages, block_table, q_start, q_lens, ctx_lens, (__nv_bfloat16*)out, part, ml, plan, rows, max_q_len, hq, hkv, ldq, ldo, max_blocks,
                         num_blocks, nsplit, scale * 1.4426950408889634f, status)) return r;
  if (nsplit == 1) return FF_HOST_OK;
  const long long joins = (nsplit ? batch * each : room.joins) * hkv * (((columns < 2 * KVT_M ? columns : 2 * KVT_M) + KVT_JOIN - 1) / KVT_JOIN);
  return launch_pdl(dim == 128 ? kv4_join_kernel<128> : kv4_join_kernel<64>, dim3((unsigned)(joins < 8 * sm_count() ? joins : 8 * sm_count())), dim3(256),
                    0, s, 0, (const float*)part, (const float2*)ml, plan, q_start, q_lens, (__nv_bfloat16*)out, batch, (int)each, rows, max_q_len, hq, hkv, ldo, nsplit);
}
