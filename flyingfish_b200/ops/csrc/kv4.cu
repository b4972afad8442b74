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

// Codes of a lane's 8 elements and the (scale, lo) of their group, which four neighbouring lanes hold together. Every lane of the warp takes part.
// ok: the group is finite and of magnitude 2^15 at most (FP16 holds what it stands for); otherwise everything is 0.
// A code comes from an FP32 quotient that is off by less than 3e-6; only where it lies within 1e-4 of a border between two codes is it taken in FP64.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[8], uint32_t& stats, bool& ok) {
  float lo = x[0], hi = x[0], big = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]);
    big = fmaxf(big, x[i] == x[i] ? fabsf(x[i]) : __uint_as_float(0x7f800000u));
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  }
  ok = big <= 32768.f;
  float scale = ok ? kv4_bf16_of_double(((double)hi - (double)lo) / 15.0) : 0.f;
  if (scale < 1.1754943508222875e-38f) scale = 0.f;          // 2^-126
  if (!ok) lo = 0.f;
  stats = pack_bf16x2(scale, lo);
  uint32_t word = 0;
  if (scale > 0.f) {
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = __fmul_rn(__fsub_rn(x[e], lo), inv);
      int c = __float2int_rn(q);
      if (fabsf(q - floorf(q) - 0.5f) < 1e-4f) c = __double2int_rn(((double)x[e] - (double)lo) / (double)scale);
      c = max(0, min(15, c));
      word |= (uint32_t)c << (4 * (e / 2 + 4 * (e & 1)));
    }
  }
  return word;
}

// Rows of packed queries, keys and values: queries and keys are RMS-normed per head (NORM) and turned (a table of cosines and sines), queries go to
// qout, keys and values into the pages of the row's slot. A head is D / 8 lanes with 8 elements each, so a turn's partner is half a head's lanes
// away and a group of 32 elements is 4 lanes. Norm and turn round as the BF16 cache's kernel does.
template <int D, bool NORM>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const __nv_bfloat16* __restrict__ qkv, const int* __restrict__ slots, uint8_t* __restrict__ kpages, uint8_t* __restrict__ vpages,
                 const float2* __restrict__ cos_sin, int rhalf, const __nv_bfloat16* __restrict__ q_weight, const __nv_bfloat16* __restrict__ k_weight,
                 float eps, __nv_bfloat16* __restrict__ qout, int rows, int hq, int hkv, long long ld, int num_blocks, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int LANES = D / 8;
  const int c = threadIdx.x & (LANES - 1);
  const int first = qout == nullptr ? hq : 0;                   // nothing to do for queries
  const int heads = hq + 2 * hkv - first;
  const long long unit = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool live = unit < (long long)rows * heads;
  const int row = live ? (int)(unit / heads) : 0, head = live ? first + (int)(unit - (long long)row * heads) : 0;
  const int part = head < hq ? 0 : (head < hq + hkv ? 1 : 2);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (live) v = reinterpret_cast<const uint4*>(qkv + (size_t)row * ld + (size_t)head * D)[c];
  float x[8];
  {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 p = unpack_bf16x2(w[i]); x[2 * i] = p.x; x[2 * i + 1] = p.y; }
  }
  if (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (part < 2) {
      const float rstd = rsqrtf(ss / (float)D + eps);
      const uint4 g = __ldg(reinterpret_cast<const uint4*>(part == 0 ? q_weight : k_weight) + c);
      const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = unpack_bf16x2(w[i]);
        x[2 * i] = kv4_bf16r(x[2 * i] * rstd * p.x);
        x[2 * i + 1] = kv4_bf16r(x[2 * i + 1] * rstd * p.y);
      }
    }
  }
  if (cos_sin != nullptr) {
    const bool upper = c >= LANES / 2;
    const int k0 = (c & (LANES / 2 - 1)) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, x[i], LANES / 2);
      if (part < 2 && k0 + i < rhalf) {
        const float2 t = cos_sin[(size_t)row * rhalf + k0 + i];
        const float a = kv4_bf16r(x[i] * t.x), b = kv4_bf16r(other * t.y);
        x[i] = kv4_bf16r(upper ? a + b : a - b);
      }
    }
  }
  if (part == 0) {
    if (live)
      reinterpret_cast<uint4*>(qout + ((size_t)row * hq + head) * D)[c] =
          make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  uint32_t stats;
  bool ok;
  const uint32_t word = kv4_quantise(x, stats, ok);             // the whole warp: its shuffles
  if (part == 0 || !live) return;
  const int slot = slots[row];
  if (slot < 0) return;
  const int block = slot / KV4_PAGE, k = slot - block * KV4_PAGE;
  if (block >= num_blocks) { if (c == 0) set_status(status, KID_KV, FF_ERR_BOUNDS, row, slot); return; }
  if (!ok && (c & 3) == 0) set_status(status, KID_KV, FF_ERR_NONFINITE, row, head);
  const int h = head - (part == 1 ? hq : hq + hkv);
  uint8_t* page = (part == 1 ? kpages : vpages) + ((size_t)block * hkv + h) * kv4_page_bytes(D);
  const int j = c >> 2, u = c & 3;
  if (part == 1) {
    reinterpret_cast<uint32_t*>(page + k * (D / 2))[u * (D / 32) + j] = word;
  } else {
    *reinterpret_cast<uint16_t*>(page + kv4_value_at<D>(k, 2 * u, j)) = (uint16_t)(word & 0xffffu);
    *reinterpret_cast<uint16_t*>(page + kv4_value_at<D>(k, 2 * u + 1, j)) = (uint16_t)(word >> 16);
  }
  if (u == 0) reinterpret_cast<uint32_t*>(page + kv4_code_bytes(D))[k * (D / 32) + j] = stats;
}

// What the pages hold for given slots, rounded to BF16; rows of a slot below 0 are zero. D / 8 lanes a head, 8 elements each.
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
// so nothing has to be sent to the device first and a captured launch keeps its own. Bound by DRAM (bytes of the pages, read and written).
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
  const long long bytes = c.bytes[blockIdx.y];
  uint8_t* const base = reinterpret_cast<uint8_t*>(c.base[blockIdx.y]);
  const uint4* src = reinterpret_cast<const uint4*>(base + bytes * c.src[blockIdx.x]);
  uint4* dst = reinterpret_cast<uint4*>(base + bytes * c.dst[blockIdx.x]);
  for (long long i = (long long)blockIdx.z * 256 + threadIdx.x; i < bytes / 16; i += (long long)gridDim.z * 256) dst[i] = src[i];
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
                  reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight)) & 15) || (reinterpret_cast<uintptr_t>(cos_sin) & 7))
    return FF_HOST_BAD_ALIGN;
  const long long units = (long long)rows * ((qout == nullptr ? 0 : hq) + 2 * hkv);
  const long long per = 256 / (dim / 8), grid = (units + per - 1) / per;
  if (grid > 0x7fffffffll) return FF_HOST_TOO_LARGE;
  auto kern = q_weight ? (dim == 128 ? kv4_write_kernel<128, true> : kv4_write_kernel<64, true>)
                       : (dim == 128 ? kv4_write_kernel<128, false> : kv4_write_kernel<64, false>);
  return launch_pdl(kern, dim3((unsigned)grid), dim3(256), 0, s, 0, (const __nv_bfloat16*)qkv, slots, (uint8_t*)kpages, (uint8_t*)vpages, (const float2*)cos_sin,
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
      const long long z = (most / 16 + 4 * 256 - 1) / (4 * 256);
      if (int r = launch_pdl(copy_pages_kernel, dim3(np, nt, (unsigned)(z < 64 ? z : 64)), dim3(256), 0, s, 0, c)) return r;
    }
  return FF_HOST_OK;
}
