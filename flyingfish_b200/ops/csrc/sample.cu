// Next tokens of a batch whose rows have settings of their own: temperature T, top-k, top-p, min-p, and one given random number u per row.
//
//   w_i = exp((l_i - max l) / T), order: logit down, id up;  kept: the first n of the order, the least of what top-k, top-p (least n whose mass
//   reaches P of the whole mass) and min-p (w_i >= min_p) leave, at least one;  drawn: lowest id whose sum of kept w up to it passes u times their sum.
//
// Ids are to be those of the formulas, so nothing that decides is rounded to 32 bits: w and its sums are FP64 (a row of 128 thousand flat tokens has
// borders 8e-6 of the mass apart, and 32-bit sums move 128 thousand of them by 1e-7 each), the histograms' masses are integers of 30 bits below the
// bin's scale, and where a border lies inside a bin its tokens are ranked one by one.
//
// A cluster of C CTAs has a row: every CTA keeps its slice of the logits in shared memory, so that they come from memory once, and a warp a run of
// consecutive ids of it. Steps, one cluster barrier each (values are pushed into every CTA's shared memory before it):
//   max; sum of w (only for top-p); histogram of the candidates over (max - l) in 1/16 octave of w, merged in CTA 0, which finds the bin that holds the
//   border; its tokens ranked in CTA 0 (bins of more than LIST tokens are divided by key first, ties of one key go by id); sums of kept w; the draw.
// Candidates: w >= (1 - P) S / V, since what lies below has less than 1 - P of the mass; w >= min_p.
//
// NaN counts as -inf, -inf is never drawn, +inf shares everything among its equals; a row without anything gives id 0 with probability 0.
#include "dtype_io.cuh"
#include "host_util.h"

namespace ff {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_CLUSTER = 8;
constexpr int SM_BINS = 1024, SM_LIST = 256, SM_TABLE = 64;

struct SampleArgs {
  const void* logits;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int* top_k;
  int* ids;
  float* probs;
  long long ld;
  int V, seg;                           // seg: ids per warp
};

struct SampleFound { int bin, count, reached; unsigned above; double mass_above; };

struct SampleShared {
  double table[SM_TABLE];               // 2^(i / 64)
  double gather[3][SM_CLUSTER];         // what every CTA of the cluster has pushed: by step
  double warp_sum[SM_WARPS];
  double scan_mass[SM_WARPS];
  double list_w[SM_LIST], sorted_w[SM_LIST];
  unsigned long long list[SM_LIST], sorted[SM_LIST];      // key << 32 | ~id
  unsigned scan_count[SM_WARPS];
  unsigned key_min[SM_CLUSTER], key_max[SM_CLUSTER];
  unsigned ties[SM_CLUSTER];
  unsigned warp_ties[SM_WARPS];
  unsigned count[SM_BINS], high[SM_BINS], low[SM_BINS];               // this CTA's: tokens, mass in digits of 15 bits
  unsigned all_count[SM_BINS], all_high[SM_BINS], all_low[SM_BINS];   // CTA 0: of the cluster, digits of 24 bits
  SampleFound found;
  unsigned border_key; int border_id;
  int list_n;
  unsigned reduce[2];
  unsigned first_id[SM_CLUSTER];
};

__device__ __forceinline__ uint32_t sm_at(const void* p, int cta) { return dsmem_addr(smem_u32(p), (uint32_t)cta); }
__device__ __forceinline__ void push_u32(const void* p, int cta, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(sm_at(p, cta)), "r"(v) : "memory"); }
__device__ __forceinline__ void push_f64(const void* p, int cta, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(sm_at(p, cta)), "d"(v) : "memory"); }
__device__ __forceinline__ void push_u64(const void* p, int cta, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sm_at(p, cta)), "l"(v) : "memory"); }
__device__ __forceinline__ void push_add(const void* p, int cta, unsigned v) { asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(sm_at(p, cta)), "r"(v) : "memory"); }
__device__ __forceinline__ unsigned push_next(const void* p, int cta) {
  unsigned r;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(r) : "r"(sm_at(p, cta)) : "memory");
  return r;
}

// keys that order as the logits do
__device__ __forceinline__ unsigned order_key(float x) { const unsigned b = __float_as_uint(x); return b & 0x80000000u ? ~b : b | 0x80000000u; }
__device__ __forceinline__ unsigned order_key(__nv_bfloat16 x) { const unsigned b = __bfloat16_as_ushort(x); return b & 0x8000u ? 0xffffu & ~b : b | 0x8000u; }
template <typename T> __device__ __forceinline__ unsigned key_of(float x);
template <> __device__ __forceinline__ unsigned key_of<float>(float x) { return order_key(x); }
template <> __device__ __forceinline__ unsigned key_of<__nv_bfloat16>(float x) { return order_key(__float2bfloat16(x)); }

template <typename T> __device__ __forceinline__ void load_vec(const T* p, float* v);
template <> __device__ __forceinline__ void load_vec<float>(const float* p, float* v) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
template <> __device__ __forceinline__ void load_vec<__nv_bfloat16>(const __nv_bfloat16* p, float* v) { load8(p, *reinterpret_cast<float(*)[8]>(v)); }

// 2^x for x <= 0, zero below 2^-1000: table of 2^(i / 64) and the Taylor polynomial of degree 4 for the rest |r| <= 1/128 (Tang, 1989); 4e-14 of the value
__device__ __forceinline__ double exp2_table(double x, const double* table) {
  if (!(x > -1000.0)) return 0.0;
  const double big = 6755399441055744.0 / 64;             // 1.5 * 2^52 / 64: the sum's last bits count 64ths
  const double s = x + big;
  const int n = __double2loint(s);
  const double r = x - (s - big);
  constexpr double L = 0.693147180559945309417;
  double p = fma(r, L * L * L * L / 24, L * L * L / 6);
  p = fma(p, r, L * L / 2);
  p = fma(p, r, L);
  p = fma(p, r, 1.0);
  p *= table[n & 63];
  return __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
}

__device__ __forceinline__ double power_of_2(int n) { return __hiloint2double((1023 + n) << 20, 0); }      // -1022 <= n <= 1023

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan64(double v, int lane) {         // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const double u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
  return v;
}
__device__ __forceinline__ unsigned warp_scan_u32(unsigned v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const unsigned u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
  return v;
}

// A row as a CTA sees it: weights and bins of its logits.
struct SampleRow {
  float top;                            // the largest logit
  double c;                             // log2(e) / T
  float bins;                           // bins per unit of logit
  const double* table;
  __device__ __forceinline__ double weight(float l) const {
    if (top == INFINITY) return l == INFINITY ? 1.0 : 0.0;
    return l == -INFINITY ? 0.0 : exp2_table(((double)l - (double)top) * c, table);
  }
  // never falls as l does: a difference and a product with a positive factor, each rounded, are monotone
  __device__ __forceinline__ int bin(float l) const {
    if (top == INFINITY) return l == INFINITY ? 0 : SM_BINS - 1;
    const float x = (top - l) * bins;
    return x < (float)(SM_BINS - 1) ? (int)x : SM_BINS - 1;
  }
};

template <typename T>
__global__ void __launch_bounds__(SM_THREADS)
sample_tokens_kernel(const SampleArgs a) {
  constexpr int VEC = 16 / sizeof(T), STEP = 32 * VEC;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  T* slice = reinterpret_cast<T*>(smem_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)(gridDim.x), rank = (int)blockIdx.x, row = blockIdx.y;
  const int per = SM_WARPS * a.seg, first = rank * per, have = max(0, min(a.V - first, per));
  const T* src = static_cast<const T*>(a.logits) + (size_t)row * a.ld + first;
  T* mine = slice + warp * a.seg;                        // this warp's ids: first + warp * seg ..
  const int id0 = first + warp * a.seg;
  cluster_arrive_relaxed();                              // "this CTA runs": waited on before the first store into a peer
  pdl_trigger();
  if (tid < SM_TABLE) sh.table[tid] = exp2(tid / 64.0);
  for (int i = tid; i < SM_BINS; i += SM_THREADS) { sh.all_count[i] = 0; sh.all_high[i] = 0; sh.all_low[i] = 0; }
  if (tid == 0) sh.list_n = 0;
  pdl_wait();

  // ---- logits into shared memory, their largest ----
  float top = -INFINITY;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  for (int i = lane * VEC; i < a.seg; i += STEP) {
    float v[VEC];
    const int at = warp * a.seg + i;
    if (vec && at + VEC <= have) {
      load_vec<T>(src + at, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = at + e < have ? to_float(src[at + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (v[e] != v[e]) v[e] = -INFINITY;
      from_float(mine + i + e, v[e]);
      top = fmaxf(top, v[e]);
    }
  }
  top = warp_max(top);
  if (lane == 0) sh.warp_sum[warp] = top;
  __syncwarp();
  cluster_wait();
  __syncthreads();
  if (tid < C) {
    double m = sh.warp_sum[0];
    for (int w = 1; w < SM_WARPS; ++w) m = fmax(m, sh.warp_sum[w]);
    push_f64(&sh.gather[0][rank], tid, m);
  }
  cluster_sync_all();
  SampleRow r;
  r.table = sh.table;
  {
    double m = sh.gather[0][0];
    for (int i = 1; i < C; ++i) m = fmax(m, sh.gather[0][i]);
    r.top = (float)m;
  }
  const float temp = a.temperature[row];
  const bool greedy = !(temp > 0.f);
  if (greedy || r.top == -INFINITY) {
    // the lowest id of the largest logit
    unsigned best = 0xffffffffu;
    for (int i = lane * VEC; i < a.seg; i += STEP) {
      float v[VEC];
      load_vec<T>(mine + i, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v[e] == r.top) best = min(best, (unsigned)(id0 + i + e));
    }
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0) sh.warp_ties[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < SM_WARPS; ++w) best = min(best, sh.warp_ties[w]);
      push_u32(&sh.first_id[rank], 0, best);
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < C; ++i) best = min(best, sh.first_id[i]);
      const bool none = r.top == -INFINITY;
      a.ids[row] = none ? 0 : (int)best;
      if (a.probs != nullptr) a.probs[row] = none ? 0.f : 1.f;
    }
    return;
  }
  r.c = 1.4426950408889634074 / (double)temp;
  r.bins = fminf((float)(r.c * 16.0), 1e30f);
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.f, floor_p = a.min_p != nullptr ? a.min_p[row] : 0.f;
  const bool use_k = k > 0 && k < a.V, use_p = p < 1.f;
  // min-p as a logit: rounded up, so that for 32-bit logits the comparison is the one with the unrounded value
  float least = -INFINITY;
  if (floor_p > 0.f && temp < INFINITY) least = r.top == INFINITY ? INFINITY : fminf(r.top, __double2float_ru((double)r.top + (double)temp * log((double)fminf(floor_p, 1.f))));

  // kept: key > border_key, or equal and id <= border_id
  unsigned border_key = 0;
  int border_id = 0x7fffffff;
  double target = 0.0;
  float cut = least;
  if (use_p) {
    double s = 0.0;
    for (int i = lane * VEC; i < a.seg; i += STEP) {
      float v[VEC];
      load_vec<T>(mine + i, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += r.weight(v[e]);
    }
    s = warp_sum64(s);
    if (lane == 0) sh.warp_sum[warp] = s;
    __syncthreads();
    if (tid < C) {
      s = sh.warp_sum[0];
      for (int w = 1; w < SM_WARPS; ++w) s += sh.warp_sum[w];
      push_f64(&sh.gather[1][rank], tid, s);
    }
    cluster_sync_all();
    s = sh.gather[1][0];
    for (int i = 1; i < C; ++i) s += sh.gather[1][i];
    target = fmax((double)p, 0.0) * s;
    if (r.top != INFINITY) {
      // borders lie at weights of (1 - P) S / V and more; a thousandth is left for the roundings
      const double away = log(0.999 * (1.0 - fmax((double)p, 0.0)) * s / a.V) * (double)temp;
      cut = fmaxf(cut, fminf(r.top, __double2float_rd((double)r.top + away)));
    }
  }
  if (use_k || use_p) {
    // ---- the border ----
    unsigned above = 0;
    double mass_above = 0.0;
    unsigned key_lo = 0, key_hi = 0xffffffffu, shift = 0;
    int bin1 = -1;
    for (int level = 0;; ++level) {
      // level 0: bins of (top - l); then the keys within the chosen bin
      __syncthreads();
      for (int i = tid; i < SM_BINS; i += SM_THREADS) { sh.count[i] = 0; sh.high[i] = 0; sh.low[i] = 0; }
      if (tid == 0) { sh.reduce[0] = 0xffffffffu; sh.reduce[1] = 0; }
      __syncthreads();
      if (level > 0) {
        unsigned lo = 0xffffffffu, hi = 0;
        for (int i = lane * VEC; i < a.seg; i += STEP) {
          float v[VEC];
          load_vec<T>(mine + i, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const unsigned key = key_of<T>(v[e]);
            if (v[e] >= cut && r.bin(v[e]) == bin1 && key >= key_lo && key <= key_hi) { lo = min(lo, key); hi = max(hi, key); }
          }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) { atomicMin(&sh.reduce[0], lo); atomicMax(&sh.reduce[1], hi); }
        __syncthreads();
        if (tid < C) { push_u32(&sh.key_min[rank], tid, sh.reduce[0]); push_u32(&sh.key_max[rank], tid, sh.reduce[1]); }
        cluster_sync_all();
        key_lo = sh.key_min[0]; key_hi = sh.key_max[0];
        for (int i = 1; i < C; ++i) { key_lo = min(key_lo, sh.key_min[i]); key_hi = max(key_hi, sh.key_max[i]); }
        if (key_lo == key_hi) break;                     // ties of one key
        shift = 0;
        while ((key_hi - key_lo) >> shift >= SM_BINS) ++shift;
      }
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (!(v[e] >= cut) || v[e] == -INFINITY) continue;
          int b = r.bin(v[e]);
          const int b1 = b;
          if (level > 0) {
            const unsigned key = key_of<T>(v[e]);
            if (b != bin1 || key < key_lo || key > key_hi) continue;
            b = (int)((key_hi - key) >> shift);
          }
          atomicAdd(&sh.count[b], 1u);
          if (use_p) {
            // mass in units of 2^-30 of the power of two above the bin's weights
            const double f = r.weight(v[e]) * power_of_2(30 + (b1 >> 4));
            const unsigned u = (unsigned)(f + 0.5);
            atomicAdd(&sh.high[b], u >> 15);
            atomicAdd(&sh.low[b], u & 32767u);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < SM_BINS; i += SM_THREADS)
        if (sh.count[i]) {
          push_add(&sh.all_count[i], 0, sh.count[i]);
          if (use_p) {
            const unsigned long long v = ((unsigned long long)sh.high[i] << 15) + sh.low[i];
            push_add(&sh.all_high[i], 0, (unsigned)(v >> 24));
            push_add(&sh.all_low[i], 0, (unsigned)(v & 0xffffffu));
          }
        }
      cluster_sync_all();
      if (rank == 0) {
        constexpr int PER = SM_BINS / SM_THREADS;
        unsigned n[PER], n_sum = 0;
        double m[PER], m_sum = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int b = tid * PER + j, b1 = level ? bin1 : b;
          n[j] = sh.all_count[b];
          m[j] = use_p ? ((double)sh.all_high[b] * 16777216.0 + (double)sh.all_low[b]) * power_of_2(-30 - (b1 >> 4)) : 0.0;
          n_sum += n[j]; m_sum += m[j];
          sh.all_count[b] = 0; sh.all_high[b] = 0; sh.all_low[b] = 0;
        }
        const unsigned n_in = warp_scan_u32(n_sum, lane);
        const double m_in = warp_scan64(m_sum, lane);
        if (lane == 31) { sh.scan_count[warp] = n_in; sh.scan_mass[warp] = m_in; }
        if (tid == 0) { sh.found.reached = 0; }
        __syncthreads();
        unsigned n_at = above + n_in - n_sum;
        double m_at = mass_above + (m_in - m_sum);
        for (int w = 0; w < warp; ++w) { n_at += sh.scan_count[w]; m_at += sh.scan_mass[w]; }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          // the first bin behind which one of the two is reached; divided bins: rounding may leave it to the last of them
          const bool before = (use_k && n_at >= (unsigned)k) || (use_p && n_at > 0 && m_at >= target);
          const bool here = (use_k && n_at + n[j] >= (unsigned)k) || (use_p && n[j] > 0 && m_at + m[j] >= target);
          if (n[j] && here && !before) { sh.found = SampleFound{tid * PER + j, (int)n[j], 1, n_at, m_at}; }
          n_at += n[j]; m_at += m[j];
        }
        __syncthreads();
        if (tid < C) {
          const SampleFound f = sh.found;
          push_u32(&sh.found.bin, tid, (unsigned)f.bin); push_u32(&sh.found.count, tid, (unsigned)f.count);
          push_u32(&sh.found.reached, tid, (unsigned)f.reached); push_u32(&sh.found.above, tid, f.above);
          push_f64(&sh.found.mass_above, tid, f.mass_above);
        }
      }
      cluster_sync_all();
      const SampleFound f = sh.found;
      if (!f.reached) {
        // level 0: no border among the candidates, min-p alone decides. A divided bin: rounding has left the border behind its last token, so the
        // whole bin is kept
        if (level > 0) border_key = key_lo;
        key_lo = 1; key_hi = 0;                          // nothing left to rank
        break;
      }
      above = f.above; mass_above = f.mass_above;
      if (level == 0) bin1 = f.bin;
      else { key_hi -= (unsigned)f.bin << shift; key_lo = max(key_lo, key_hi - ((1u << shift) - 1)); }
      if (f.count <= SM_LIST) break;
    }
    if (key_lo == key_hi && sh.found.count > SM_LIST) {
      // ---- ties of one key: as many of the lowest ids as are needed ----
      unsigned n = 0;
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) n += key_of<T>(v[e]) == key_lo && v[e] >= cut;
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sh.warp_ties[warp] = n;
      __syncthreads();
      unsigned in_cta = 0;
      for (int w = 0; w < SM_WARPS; ++w) in_cta += sh.warp_ties[w];
      if (tid < C) push_u32(&sh.ties[rank], tid, in_cta);
      cluster_sync_all();
      unsigned all = 0, before = 0;
      for (int i = 0; i < C; ++i) { if (i < rank) before += sh.ties[i]; all += sh.ties[i]; }
      unsigned want = all;
      if (use_k) want = min(want, (unsigned)k - above);
      if (use_p) {
        const float l = sizeof(T) == 2 ? __bfloat162float(__ushort_as_bfloat16((unsigned short)(key_lo & 0x8000u ? key_lo & 0x7fffu : ~key_lo)))
                                       : __uint_as_float(key_lo & 0x80000000u ? key_lo & 0x7fffffffu : ~key_lo);
        const double need = ceil((target - mass_above) / r.weight(l));
        if (need < (double)want) want = need < 1.0 ? 1u : (unsigned)need;
      }
      for (int w = 0; w < warp; ++w) before += sh.warp_ties[w];
      if (want > before && want <= before + n) {         // this warp holds the last one
        unsigned at = before;
        for (int i = lane * VEC; i - lane * VEC < a.seg; i += STEP) {
          float v[VEC];
          unsigned here = 0;
          load_vec<T>(mine + i, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) here += key_of<T>(v[e]) == key_lo && v[e] >= cut;
          const unsigned upto = warp_scan_u32(here, lane);
          unsigned seen = at + upto - here;
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (key_of<T>(v[e]) == key_lo && v[e] >= cut && ++seen == want)
              for (int t = 0; t < C; ++t) push_u32(&sh.border_id, t, (unsigned)(id0 + i + e));
          at += __shfl_sync(0xffffffffu, upto, 31);
        }
      }
      cluster_sync_all();
      border_key = key_lo; border_id = sh.border_id;
    } else if (key_lo <= key_hi) {
      // ---- few tokens: ranked one by one in CTA 0 ----
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const unsigned key = key_of<T>(v[e]);
          if (!(v[e] >= cut) || v[e] == -INFINITY || r.bin(v[e]) != bin1 || key < key_lo || key > key_hi) continue;
          const unsigned slot = push_next(&sh.list_n, 0);
          if (slot < SM_LIST) {
            push_u64(&sh.list[slot], 0, (unsigned long long)key << 32 | (unsigned)~(id0 + i + e));
            push_f64(&sh.list_w[slot], 0, use_p ? r.weight(v[e]) : 0.0);
          }
        }
      }
      cluster_sync_all();
      if (rank == 0) {
        const int n = min(sh.list_n, SM_LIST);
        if (tid < n) {
          const unsigned long long me = sh.list[tid];
          int at = 0;
          for (int j = 0; j < n; ++j) at += sh.list[j] > me;
          sh.sorted[at] = me; sh.sorted_w[at] = sh.list_w[tid];
        }
        __syncthreads();
        double w = tid < n ? sh.sorted_w[tid] : 0.0;
        const double upto = warp_scan64(w, lane);
        if (lane == 31) sh.scan_mass[warp] = upto;
        __syncthreads();
        double m = mass_above + upto;
        for (int i = 0; i < warp; ++i) m += sh.scan_mass[i];
        bool here = tid < n && ((use_k && above + tid + 1 >= (unsigned)k) || (use_p && m >= target));
        here = here || tid == n - 1;
        // the first of them
        const unsigned vote = __ballot_sync(0xffffffffu, here);
        if (lane == 0) sh.scan_count[warp] = vote ? (unsigned)(warp * 32 + __ffs(vote) - 1) : 0xffffffffu;
        __syncthreads();
        if (tid < C) {
          unsigned at = 0xffffffffu;
          for (int i = 0; i < SM_WARPS; ++i) at = min(at, sh.scan_count[i]);
          const unsigned long long border = sh.sorted[at];
          push_u32(&sh.border_key, tid, (unsigned)(border >> 32));
          push_u32(&sh.border_id, tid, ~(unsigned)border);
        }
      }
      cluster_sync_all();
      border_key = sh.border_key; border_id = sh.border_id;
    }
  }

  // ---- sums of the kept weights, and the draw ----
  auto kept = [&](float l, int id) {
    const unsigned key = key_of<T>(l);
    return l >= least && (key > border_key || (key == border_key && id <= border_id));
  };
  double s = 0.0;
  for (int i = lane * VEC; i < a.seg; i += STEP) {
    float v[VEC];
    load_vec<T>(mine + i, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (kept(v[e], id0 + i + e)) s += r.weight(v[e]);
  }
  s = warp_sum64(s);
  __syncthreads();
  if (lane == 0) sh.warp_sum[warp] = s;
  __syncthreads();
  if (tid < C) {
    double t = sh.warp_sum[0];
    for (int w = 1; w < SM_WARPS; ++w) t += sh.warp_sum[w];
    push_f64(&sh.gather[2][rank], tid, t);
  }
  cluster_sync_all();
  double all = 0.0, before = 0.0;
  int last = 0;                                          // the last CTA that holds any of the mass
  for (int i = 0; i < C; ++i) { if (i == rank) before = all; all += sh.gather[2][i]; if (sh.gather[2][i] > 0.0) last = i; }
  float u = a.uniforms[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  const double goal = (double)u * all;
  double after = before + sh.gather[2][rank];
  if (!(goal >= before && (goal < after || rank == last) && sh.gather[2][rank] > 0.0)) return;
  // this CTA has it: the warp, then the token
  int last_warp = 0;
  double at = before, from = before;
  for (int w = 0; w < SM_WARPS; ++w) { if (w == warp) from = at; at += sh.warp_sum[w]; if (sh.warp_sum[w] > 0.0) last_warp = w; }
  const double mass = sh.warp_sum[warp];
  // the warps' ends as every warp computes them: from + mass is the next one's `from`
  if (!(mass > 0.0 && goal >= from && (goal < from + mass || warp == last_warp))) return;
  int pick = -1, spare = -1;
  double pick_w = 0.0, spare_w = 0.0;
  for (int i0 = 0; i0 < a.seg && pick < 0; i0 += STEP) {
    const int i = i0 + lane * VEC;
    float v[VEC];
    load_vec<T>(mine + i, v);
    double w[VEC], sum = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) { w[e] = kept(v[e], id0 + i + e) ? r.weight(v[e]) : 0.0; sum += w[e]; }
    const double upto = warp_scan64(sum, lane);
    double x = from + (upto - sum);
    int got = -1, some = -1;
    double got_w = 0.0, some_w = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      x += w[e];
      if (w[e] > 0.0) {
        some = id0 + i + e; some_w = w[e];
        if (got < 0 && x > goal) { got = some; got_w = w[e]; }
      }
    }
    const unsigned vote = __ballot_sync(0xffffffffu, got >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
    if (vote) {
      pick = __shfl_sync(0xffffffffu, got, __ffs(vote) - 1);
      pick_w = __shfl_sync(0xffffffffu, got_w, __ffs(vote) - 1);
    }
    if (any) {
      spare = __shfl_sync(0xffffffffu, some, 31 - __clz(any));
      spare_w = __shfl_sync(0xffffffffu, some_w, 31 - __clz(any));
    }
    from += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (pick < 0) { pick = spare; pick_w = spare_w; }      // the sums' last bits left the goal behind the last token
  if (lane == 0) {
    a.ids[row] = pick;
    if (a.probs != nullptr) a.probs[row] = (float)(pick_w / all);
  }
}

}  // namespace ff
using namespace ff;

template <typename T>
static int sample_launch(const SampleArgs& args, int rows, cudaStream_t stream) {
  constexpr int STEP = 32 * (16 / (int)sizeof(T)), MOST = 227 * 1024;
  const int fixed = ((int)sizeof(SampleShared) + 15) / 16 * 16;
  SampleArgs a = args;
  int c = 8;
  while (c > 1 && (long long)rows * c > 444 && (long long)(a.V + c / 2 - 1) / (c / 2) * sizeof(T) + fixed + 16 * STEP * sizeof(T) <= MOST) c /= 2;
  a.seg = (a.V + c * SM_WARPS - 1) / (c * SM_WARPS);
  a.seg = (a.seg + STEP - 1) / STEP * STEP;
  const long long smem = fixed + (long long)SM_WARPS * a.seg * sizeof(T);
  if (smem > MOST || rows > 65535) return FF_HOST_TOO_LARGE;
  auto kern = sample_tokens_kernel<T>;
  if (int e = opt_in_smem(kern, (int)smem)) return e;
  return launch_pdl(kern, dim3(c, rows), dim3(SM_THREADS), (size_t)smem, stream, c, a);
}

// logits [rows, V] BF16 (fp32 = 0) or FP32, pitch ld; uniforms, temperature [rows]; top_k, top_p, min_p [rows] or null; ids [rows], probs [rows] or null.
FF_EXPORT int ff_sample_tokens(const void* logits, int fp32, const float* uniforms, const float* temperature, const int* top_k, const float* top_p,
                               const float* min_p, int* ids, float* probs, int rows, int V, long long ld, cudaStream_t stream) {
  if (rows <= 0 || V <= 0 || ld < 0 || logits == nullptr || uniforms == nullptr || temperature == nullptr || ids == nullptr) return FF_HOST_BAD_SHAPE;
  const SampleArgs a = {logits, uniforms, temperature, top_p, min_p, top_k, ids, probs, ld, V, 0};
  return fp32 ? sample_launch<float>(a, rows, stream) : sample_launch<__nv_bfloat16>(a, rows, stream);
}
