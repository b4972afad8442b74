// Writing, reading back and copying pages of the 4-bit key / value cache (layout and format: kv4.cuh).
#include "kv4.cuh"
#include "host_util.h"

namespace ff {

__device__ __forceinline__ float kv4_bf16r(float x) { return __bfloat162float(__float2bfloat16(x)); }

// RN_bf16(x) of a double with one rounding: to FP32 by truncation with the rest kept in the last bit (24 bits are far more than
// the 8 + 2 that make the second rounding the only one), then to BF16.
__device__ __forceinline__ float kv4_bf16_of_double(double x) {
  float f = __double2float_rz(x);
  if ((double)f != x) f = __uint_as_float(__float_as_uint(f) | 1u);
  return kv4_bf16r(f);
}

__device__ __forceinline__ uint32_t kv4_add2(uint32_t a, uint32_t b) { uint32_t r; asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t kv4_min2(uint32_t a, uint32_t b) { uint32_t r; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t kv4_max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }

// Codes of a lane's 8 elements (w: BF16 pairs) and the (scale, lo) of their group, which four neighbouring lanes hold together. Every lane of the warp takes part.
// ok: the group is finite and of magnitude 2^15 at most (FP16 holds what it stands for); otherwise everything is 0.
// A code comes from an FP32 quotient that is off by less than 3e-6; only where one lies within 1e-4 of a border between two codes are they taken in FP64.
__device__ __forceinline__ uint32_t kv4_quantise(const uint32_t (&w)[4], uint32_t& stats, bool& ok) {
  uint32_t mn = kv4_min2(kv4_min2(w[0], w[1]), kv4_min2(w[2], w[3])), mx = kv4_max2(kv4_max2(w[0], w[1]), kv4_max2(w[2], w[3]));
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    mn = kv4_min2(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = kv4_max2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  mn = kv4_min2(mn, mn >> 16); mx = kv4_max2(mx, mx >> 16);     // (the lower half counts)
  float lo = __uint_as_float(mn << 16) + 0.f;                    // (no negative zero)
  const float hi = __uint_as_float(mx << 16);
  ok = lo >= -32768.f && hi <= 32768.f;                          // false where one of them is no number
  // the scale: an FP32 quotient, off by less than 2^-22 of it, whose rounding to BF16 is in doubt only next to the middle between two BF16 numbers
  float scale = __fmul_rn(__fsub_rn(hi, lo), 0.0666666667f);
  const uint32_t low = __float_as_uint(scale) & 0xffffu;
  if (low - 0x7ff0u <= 0x20u) scale = kv4_bf16_of_double(((double)hi - (double)lo) / 15.0);
  else scale = kv4_bf16r(scale);
  if (!ok) { scale = 0.f; lo = 0.f; }
  if (scale < 1.1754943508222875e-38f) scale = 0.f;              // 2^-126
  stats = pack_bf16x2(scale, lo);
  if (!(scale > 0.f)) return 0u;
  // codes: q + 3 2^22 has the integer next to q in its last bits, of which those of a word are summed; what the upper bits add is known
  const float inv = __frcp_rn(scale);
  uint32_t word = 0u - (0x4b400000u + 0xb4000000u + 0x40000000u);
  uint32_t doubt = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    const float q = __fmul_rn(__fsub_rn(x, lo), inv), r = __fadd_rn(q, 12582912.f);
    if (fabsf(__fsub_rn(q, __fsub_rn(r, 12582912.f))) > 0.4999f) doubt |= 1u << e;
    word += __float_as_uint(r) << (4 * (e / 2 + 4 * (e & 1)));
  }
  if (doubt) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (doubt >> e & 1u) {
        const float x = __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        const int at = 4 * (e / 2 + 4 * (e & 1));
        word = (word & ~(15u << at)) | ((uint32_t)min(15, __double2int_rn(((double)x - (double)lo) / (double)scale)) << at);
      }
  }
  return word;
}

// Rows of packed queries, keys and values: queries and keys are RMS-normed per head (NORM) and turned (a table of cosines and sines), queries go to
// qout, keys and values into the pages of the row's slot. A head is D / 8 lanes with 8 elements each, so a turn's partner is half a head's lanes
// away and a group of 32 elements is 4 lanes; such a set of lanes walks heads of a row with the row's cosines and sines in registers, five heads on their way at
// once. Norm and turn round as the BF16 cache's kernel does: every product and sum to BF16 (packed instructions; a sum of two BF16 numbers that FP32 does not
// hold has a term too small to matter). Few rows are spread over CTAs by heads. 8191 rows of 64 + 2 x 8 heads of 128: 78 us, 4.2 TB/s, where the bytes alone take 50: issue
// slots are 63 % taken, warps wait for their loads in between. With FP64 for all codes of a lane that has one in doubt (a third of the warps have) 82, with three
// heads at once 102, with 80 registers and three CTAs 90. Five heads at once are 80 heads in one round of 16 sets of lanes; other numbers lose up to 7 % by it: 48 heads 65 us where three at
// once take 62, 10 heads 43 and 40, 36 of 64 elements 45 and 44, 96 heads 138 and 132.
constexpr int WRITE_THREADS = 256, WRITE_HEADS = 5;
template <int D, bool NORM>
__global__ void __launch_bounds__(WRITE_THREADS, 4)
kv4_write_kernel(const __nv_bfloat16* __restrict__ qkv, const int* __restrict__ slots, uint8_t* __restrict__ kpages, uint8_t* __restrict__ vpages,
                 const float2* __restrict__ cos_sin, int rhalf, const __nv_bfloat16* __restrict__ q_weight, const __nv_bfloat16* __restrict__ k_weight,
                 float eps, __nv_bfloat16* __restrict__ qout, int rows, int hq, int hkv, long long ld, int num_blocks, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int LANES = D / 8, SETS = WRITE_THREADS / LANES;
  const int c = threadIdx.x & (LANES - 1);
  const int first = qout == nullptr ? hq : 0, heads = hq + 2 * hkv;               // nothing to do for queries?
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const int slot = slots[row];
    const int block = slot / KV4_PAGE, k = slot - block * KV4_PAGE;
    if (slot >= 0 && block >= num_blocks && threadIdx.x == 0) set_status(status, KID_KV, FF_ERR_BOUNDS, row, slot);
    const bool store = slot >= 0 && block < num_blocks, upper = c >= LANES / 2, turn = cos_sin != nullptr, whole = 2 * rhalf == D;
    uint32_t cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { cs[i] = 0x3f803f80u; sn[i] = 0u; }
    if (turn) {
      // elements of a head's halves from rhalf on stay: cosine 1, sine 0 would give x + 0, which is x but for a zero's sign
      const int k0 = (c & (LANES / 2 - 1)) * 8;
      float x[8], y[8];
      const float2* table = cos_sin + (size_t)row * rhalf + k0;
      if (k0 + 8 <= rhalf && (rhalf & 1) == 0) {                     // (even rows of a 16-byte aligned table)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 t = reinterpret_cast<const float4*>(table)[i];
          x[2 * i] = t.x; y[2 * i] = t.y; x[2 * i + 1] = t.z; y[2 * i + 1] = t.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 t = k0 + i < rhalf ? table[i] : make_float2(1.f, 0.f);
          x[i] = t.x; y[i] = t.y;
        }
      }
      if (!upper) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = -y[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { cs[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]); sn[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]); }
    }
    const int stays = rhalf - (c & (LANES / 2 - 1)) * 8;                             // elements of the lane from here on do not turn
    const __nv_bfloat16* const in = qkv + (size_t)row * ld + c * 8;
    __nv_bfloat16* const qo = qout + (size_t)row * hq * D + c * 8;
    const int set = blockIdx.y * SETS + threadIdx.x / LANES, step = gridDim.y * SETS;
    for (int base = first + set; base - set < heads; base += WRITE_HEADS * step) {   // the same number of rounds for every lane of a warp
      uint4 v[WRITE_HEADS];
#pragma unroll
      for (int u = 0; u < WRITE_HEADS; ++u) {
        const int head = base + u * step;
        v[u] = make_uint4(0, 0, 0, 0);
        if (head < heads) v[u] = *reinterpret_cast<const uint4*>(in + head * D);
      }
#pragma unroll
      for (int u = 0; u < WRITE_HEADS; ++u) {
        const int head = base + u * step;
        if (base - set + u * step >= heads) break;                                   // (for all lanes)
        const int part = head < hq ? 0 : (head < hq + hkv ? 1 : 2);
        const bool live = head < heads;
        uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        if (NORM) {
          float x[8], ss = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) { const float2 p = unpack_bf16x2(w[i]); x[2 * i] = p.x; x[2 * i + 1] = p.y; ss += p.x * p.x + p.y * p.y; }
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (part < 2) {
            const float rstd = rsqrtf(ss / (float)D + eps);
            const uint4 g = __ldg(reinterpret_cast<const uint4*>(part == 0 ? q_weight : k_weight) + c);
            const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float2 p = unpack_bf16x2(gw[i]); w[i] = pack_bf16x2(x[2 * i] * rstd * p.x, x[2 * i + 1] * rstd * p.y); }
          }
        }
        if (turn) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, w[i], LANES / 2);
            const uint32_t t = kv4_add2(kv4_mul2(w[i], cs[i]), kv4_mul2(other, sn[i]));
            if (whole) {
              if (part < 2) w[i] = t;
            } else {
              const uint32_t keep = 2 * i >= stays ? 0xffffffffu : 2 * i + 1 >= stays ? 0xffff0000u : 0u;
              if (part < 2) w[i] = (t & ~keep) | (w[i] & keep);
            }
          }
        }
        if (part == 0 && live && qout != nullptr) *reinterpret_cast<uint4*>(qo + head * D) = make_uint4(w[0], w[1], w[2], w[3]);
        const bool mine = part > 0 && live && store;
        if (__any_sync(0xffffffffu, mine)) {
          uint32_t stats;
          bool ok;
          const uint32_t word = kv4_quantise(w, stats, ok);
          if (mine) {
            if (!ok && (c & 3) == 0) set_status(status, KID_KV, FF_ERR_NONFINITE, row, head);
            const int h = head - (part == 1 ? hq : hq + hkv);
            uint8_t* page = (part == 1 ? kpages : vpages) + ((size_t)block * hkv + h) * kv4_page_bytes(D);
            const int j = c >> 2, y = c & 3;
            if (part == 1) {
              reinterpret_cast<uint32_t*>(page + k * (D / 2))[y * (D / 32) + j] = word;
            } else {
              *reinterpret_cast<uint16_t*>(page + kv4_value_at<D>(k, 2 * y, j)) = (uint16_t)(word & 0xffffu);
              *reinterpret_cast<uint16_t*>(page + kv4_value_at<D>(k, 2 * y + 1, j)) = (uint16_t)(word >> 16);
            }
            if (y == 0) reinterpret_cast<uint32_t*>(page + kv4_code_bytes(D))[k * (D / 32) + j] = stats;
          }
        }
      }
    }
  }
}

// What the pages hold for given slots, rounded to BF16; rows of a slot below 0 are zero. D / 8 lanes a head, 8 elements each. The 8191 rows above, 34 MB of
// results from 21 MB of pages: 23 us with its launch, where the bytes take 8: a thread makes one 16-byte result and has nothing else in flight, and values come as two 16-bit loads.
template <int D>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ kpages, const uint8_t* __restrict__ vpages, const int* __restrict__ slots, __nv_bfloat16* __restrict__ kout,
                __nv_bfloat16* __restrict__ vout, int rows, int hkv, int num_blocks, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int LANES = D / 8;
  const long long unit = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (unit >= (long long)rows * 2 * hkv) return;
  const int c = threadIdx.x & (LANES - 1), row = (int)(unit / (2 * hkv)), h2 = (int)(unit - (long long)row * 2 * hkv);
  const bool keys = h2 < hkv;
  const int h = keys ? h2 : h2 - hkv;
  const int slot = slots[row];
  uint4 out = make_uint4(0, 0, 0, 0);
  const int block = slot / KV4_PAGE, k = slot - block * KV4_PAGE;
  if (slot >= 0 && block >= num_blocks) { if (c == 0) set_status(status, KID_KV, FF_ERR_BOUNDS, row, slot); }
  else if (slot >= 0) {
    const uint8_t* page = (keys ? kpages : vpages) + ((size_t)block * hkv + h) * kv4_page_bytes(D);
    const int j = c >> 2, u = c & 3;
    const uint32_t word = keys ? reinterpret_cast<const uint32_t*>(page + k * (D / 2))[u * (D / 32) + j]
                               : (uint32_t)*reinterpret_cast<const uint16_t*>(page + kv4_value_at<D>(k, 2 * u, j)) |
                                     (uint32_t)*reinterpret_cast<const uint16_t*>(page + kv4_value_at<D>(k, 2 * u + 1, j)) << 16;
    const float2 st = unpack_bf16x2(reinterpret_cast<const uint32_t*>(page + kv4_code_bytes(D))[k * (D / 32) + j]);
    uint32_t* w = &out.x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = pack_bf16x2(fmaf((float)((word >> (4 * i)) & 15u), st.x, st.y), fmaf((float)((word >> (4 * i + 16)) & 15u), st.x, st.y));
  }
  reinterpret_cast<uint4*>((keys ? kout : vout) + ((size_t)row * hkv + h) * D)[c] = out;
}

// Pages copied inside every tensor of a list: one launch for all layers' keys and values. Addresses and page numbers are arguments of the launch,
// so nothing has to be sent to the device first and a captured launch keeps its own. Bound by DRAM: 150 BF16 blocks in 32 layers, 2.5 GB read and written, 396 us where a
// plain copy's rate gives 383. A single page of 32 layers is bound by its 64 tensors' addresses on the host, 47 us.
constexpr int COPY_TENSORS = 160, COPY_PAIRS = 256;
struct CopyPages {
  unsigned long long base[COPY_TENSORS];
  unsigned bytes[COPY_TENSORS];              // of a page
  int src[COPY_PAIRS], dst[COPY_PAIRS];
};
static_assert(sizeof(CopyPages) <= 4064, "arguments of a launch");

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyPages c) {
  pdl_trigger();
  pdl_wait();
  const long long n = c.bytes[blockIdx.y] / 16;
  uint8_t* const base = reinterpret_cast<uint8_t*>(c.base[blockIdx.y]);
  const uint4* src = reinterpret_cast<const uint4*>(base) + n * c.src[blockIdx.x];
  uint4* dst = reinterpret_cast<uint4*>(base) + n * c.dst[blockIdx.x];
  for (long long i0 = (long long)blockIdx.z * 1024 + threadIdx.x; i0 < n; i0 += (long long)gridDim.z * 1024) {
    uint4 v[4];                                      // four on their way at once (one at a time: 485 us for 2.5 GB)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < n) v[u] = __ldcs(src + i0 + u * 256);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < n) __stcs(dst + i0 + u * 256, v[u]);
  }
}

}  // namespace ff
using namespace ff;

// qkv rows [rows, ld] of hq + 2 hkv heads of dim elements; slots int32 [rows]; pages [num_blocks, hkv, page bytes]. cos_sin: float2 [rows, rhalf] or null;
// q_weight / k_weight: [dim] or both null; qout [rows, hq dim] or null (queries stay as they are: neither table nor weights may be given).
FF_EXPORT int ff_kv4_write(const void* qkv, const int* slots, void* kpages, void* vpages, const void* cos_sin, int rhalf, const void* q_weight,
                           const void* k_weight, float eps, void* qout, int rows, int hq, int hkv, int dim, long long ld, int num_blocks, int* status,
                           cudaStream_t s) {
  if (rows <= 0 || hq <= 0 || hkv <= 0 || (dim != 64 && dim != 128) || num_blocks <= 0) return FF_HOST_BAD_SHAPE;
  if (ld < (long long)(hq + 2 * hkv) * dim || rhalf < 0 || rhalf > dim / 2) return FF_HOST_BAD_SHAPE;
  if ((q_weight == nullptr) != (k_weight == nullptr) || (qout == nullptr && (cos_sin != nullptr || q_weight != nullptr))) return FF_HOST_BAD_SHAPE;
  if (ld % 8 || ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(kpages) | reinterpret_cast<uintptr_t>(vpages) | reinterpret_cast<uintptr_t>(qout) |
                  reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight)) & 15) || (reinterpret_cast<uintptr_t>(cos_sin) & 15))
    return FF_HOST_BAD_ALIGN;
  const int sets = WRITE_THREADS / (dim / 8), heads = (qout == nullptr ? 0 : hq) + 2 * hkv;
  // few rows: a CTA for every set of heads that its lanes take at once; many: a row's heads in one, whose loads are on their way together
  const int at_once = rows >= 4 * sm_count() ? sets * WRITE_HEADS : sets, y = (heads + at_once - 1) / at_once;
  if (y > 65535) return FF_HOST_TOO_LARGE;
  auto kern = q_weight ? (dim == 128 ? kv4_write_kernel<128, true> : kv4_write_kernel<64, true>)
                       : (dim == 128 ? kv4_write_kernel<128, false> : kv4_write_kernel<64, false>);
  return launch_pdl(kern, dim3((unsigned)(rows < 16 * sm_count() ? rows : 16 * sm_count()), y), dim3(WRITE_THREADS), 0, s, 0, (const __nv_bfloat16*)qkv, slots, (uint8_t*)kpages, (uint8_t*)vpages, (const float2*)cos_sin,
                    rhalf, (const __nv_bfloat16*)q_weight, (const __nv_bfloat16*)k_weight, eps, (__nv_bfloat16*)qout, rows, hq, hkv, ld, num_blocks, status);
}

FF_EXPORT int ff_kv4_read(const void* kpages, const void* vpages, const int* slots, void* kout, void* vout, int rows, int hkv, int dim, int num_blocks,
                          int* status, cudaStream_t s) {
  if (rows <= 0 || hkv <= 0 || (dim != 64 && dim != 128) || num_blocks <= 0) return FF_HOST_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(kpages) | reinterpret_cast<uintptr_t>(vpages) | reinterpret_cast<uintptr_t>(kout) | reinterpret_cast<uintptr_t>(vout)) & 15)
    return FF_HOST_BAD_ALIGN;
  const long long per = 256 / (dim / 8), grid = ((long long)rows * 2 * hkv + per - 1) / per;
  if (grid > 0x7fffffffll) return FF_HOST_TOO_LARGE;
  return launch_pdl(dim == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>, dim3((unsigned)grid), dim3(256), 0, s, 0, (const uint8_t*)kpages, (const uint8_t*)vpages,
                    slots, (__nv_bfloat16*)kout, (__nv_bfloat16*)vout, rows, hkv, num_blocks, status);
}

// base / bytes: host arrays, one entry per tensor; src / dst: host arrays of page numbers, no page of dst twice or in src.
FF_EXPORT int ff_copy_pages(const unsigned long long* base, const long long* bytes, int tensors, const int* src, const int* dst, int pairs, cudaStream_t s) {
  if (tensors <= 0 || pairs <= 0) return FF_HOST_BAD_SHAPE;
  for (int t = 0; t < tensors; ++t) {
    if (bytes[t] <= 0 || bytes[t] > 0x7fffffffll) return FF_HOST_BAD_SHAPE;
    if ((base[t] & 15) || (bytes[t] & 15)) return FF_HOST_BAD_ALIGN;
  }
  for (int t0 = 0; t0 < tensors; t0 += COPY_TENSORS)
    for (int p0 = 0; p0 < pairs; p0 += COPY_PAIRS) {
      CopyPages c;
      const int nt = tensors - t0 < COPY_TENSORS ? tensors - t0 : COPY_TENSORS, np = pairs - p0 < COPY_PAIRS ? pairs - p0 : COPY_PAIRS;
      long long most = 0;
      for (int t = 0; t < nt; ++t) { c.base[t] = base[t0 + t]; c.bytes[t] = (unsigned)bytes[t0 + t]; most = bytes[t0 + t] > most ? bytes[t0 + t] : most; }
      for (int p = 0; p < np; ++p) { c.src[p] = src[p0 + p]; c.dst[p] = dst[p0 + p]; }
      const long long z = (most / 16 + 1023) / 1024;
      if (int r = launch_pdl(copy_pages_kernel, dim3(np, nt, (unsigned)(z < 64 ? z : 64)), dim3(256), 0, s, 0, c)) return r;
    }
  return FF_HOST_OK;
}
