// Next tokens of a batch whose rows have settings of their own: temperature T, top-k, top-p, min-p, and one given random number u per row.
//
//   w_i = exp((l_i - max l) / T), order: logit down, id up;  kept: the first n of the order, the least of what top-k, top-p (least n whose mass
//   reaches P of the whole mass) and min-p (w_i >= min_p) leave, at least one;  drawn: lowest id whose sum of kept w up to it passes u times their sum.
//
// Ids are to be those of the formulas, so what decides is held in FP64: a row of 128 thousand flat tokens has borders 8e-6 of the mass apart, and
// 32-bit sums move 128 thousand of them by 1e-7 each. Less than FP64 has are the weights (1.2e-12 of themselves, exp2_table) and, where a list is joined with
// the masses in front of it, the list's (multiples of 2^-50 of the largest weight): a millionth of the distance of those borders.
//
// A cluster of C CTAs has a row: every CTA keeps its slice of the logits in shared memory, so that they come from memory once, and a warp a run of
// consecutive ids of it. Values cross by stores into the peers' shared memory in front of a cluster barrier. Steps:
//   1 the largest logit;
//   2 the mass, where top-p or the draw needs it, and a logit that at least k tokens reach, where top-k is on: of a CTA's threads' largest logits the n-th,
//     n its share of k, the least over the CTAs;
//   3 without top-k and top-p: the draw. Else the candidates -- logits at or above what top-k leaves, (1 - P) S / V (less has less than 1 - P of the
//     mass) and min-p -- go to CTA 0, which sorts them, finds the border, sorts the kept ones by id and draws;
//   4 more than SM_LIST candidates (flat rows): a histogram of the candidates' logits, masses in 14 bits, says in which bin the border lies, or two if it
//     cannot tell; the mass above is summed in FP64 and the bin's tokens are sorted as in 3. A bin of more tokens is divided by key, ties of one key go by
//     id. CTA 0 finds the warp whose run holds the draw, and that warp's CTA the token.
//
// What bounds it: dependent steps, each with a barrier of the cluster, in small batches (one flat row of 128256: 25 us, 33 rows of 50257 with top-k 17);
// issue slots in large ones (256 rows of 151936 with top-k, top-p and min-p: 87 us, 57 % of the slots, FP64 pipe 27 %, 0.9 TB/s). Why shared memory: the
// logits are looked at three to six times. Why FP64 and no compensated FP32: an SM has half as many FP64 lanes, and pairs of words take more than twice the operations.
//
// NaN counts as -inf, -inf is never drawn, +inf shares everything among its equals; a row without anything gives id 0 with probability 0.
#include "dtype_io.cuh"
#include "host_util.h"

namespace ff {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_CLUSTER = 8;
constexpr int SM_BINS = 1024, SM_LIST = 1024, SM_SMALL = 128, SM_TABLE = 32, SM_COPIES = 16, SM_PARTS = SM_CLUSTER * SM_WARPS;
constexpr int SM_MOST_SMEM = 227 * 1024, SM_STEP_BYTES = 512, SM_MOST_STEPS = 32;        // most steps of a warp's run: one per lane where the draw looks for the step
constexpr float SM_FAR = -1000.f;       // octaves below the largest from which on a token weighs nothing

struct SampleArgs {
  const void* logits;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int* top_k;
  int* ids;
  float* probs;
  long long ld;
  int V, seg;                           // seg: ids per warp
};

struct SampleFound { int lo, hi, count; unsigned above; };

struct SampleShared {
  double table[SM_TABLE * SM_COPIES];   // 2^(i / 32), every lane of a half warp its own
  double mass[SM_CLUSTER];              // what every CTA of the cluster has pushed: the mass
  double part[SM_PARTS];                // CTA 0, general path: every warp's kept mass in front of the border's bins
  unsigned part_in[SM_PARTS][3];        // and within them, whole numbers of 2^-10, 2^-30 and 2^-50, so that the order of their sum does not matter
  double warp_sum[SM_WARPS], scan_mass[SM_WARPS];
  double total, from, c, below;
  float top[SM_CLUSTER], cut[SM_CLUSTER], warp_top[SM_WARPS];
  int candidates[SM_CLUSTER];
  unsigned key_min[SM_CLUSTER], key_max[SM_CLUSTER], ties[SM_CLUSTER], first_id[SM_CLUSTER];
  unsigned warp_ties[SM_WARPS], scan_count[SM_WARPS];
  unsigned reduce[2];
  SampleFound found;
  unsigned border_key;
  int border_id, list_n, at, owner;
  double step_sum[SM_MOST_STEPS];       // mass of each step of the run that holds the draw
  union {
    struct {                            // a list of tokens: key << 32 | ~id, and their weights; where the bins of a sort begin
      unsigned long long list[SM_LIST];
      double w[SM_LIST];
      unsigned place[SM_LIST + 1];
    };
    struct {                            // histogram: this CTA's, and in CTA 0 the cluster's
      unsigned count[SM_BINS], mass_of[SM_BINS];
      unsigned all_count[SM_BINS], all_high[SM_BINS], all_low[SM_BINS];
    };
  };
};

__device__ __forceinline__ uint32_t sm_at(const void* p, int cta) { return dsmem_addr(smem_u32(p), (uint32_t)cta); }
__device__ __forceinline__ void push_u32(const void* p, int cta, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(sm_at(p, cta)), "r"(v) : "memory"); }
__device__ __forceinline__ void push_f64(const void* p, int cta, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(sm_at(p, cta)), "d"(v) : "memory"); }
__device__ __forceinline__ void push_u64(const void* p, int cta, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sm_at(p, cta)), "l"(v) : "memory"); }
__device__ __forceinline__ void push_add(const void* p, int cta, unsigned v) { asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(sm_at(p, cta)), "r"(v) : "memory"); }
__device__ __forceinline__ unsigned push_take(const void* p, int cta, unsigned n) {
  unsigned r;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(sm_at(p, cta)), "r"(n) : "memory");
  return r;
}

// keys that order as the logits do, zeros of both signs as one: BF16 values have the upper half of an FP32 key
__device__ __forceinline__ unsigned order_key(float x) { const unsigned b = __float_as_uint(x + 0.f); return b & 0x80000000u ? ~b : b | 0x80000000u; }
template <typename T> __device__ __forceinline__ unsigned key_of(float x) { return order_key(x) >> (sizeof(T) == 2 ? 16 : 0); }

template <typename T> __device__ __forceinline__ float logit_of(unsigned key);
template <> __device__ __forceinline__ float logit_of<float>(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
template <> __device__ __forceinline__ float logit_of<__nv_bfloat16>(unsigned key) {
  return __bfloat162float(__ushort_as_bfloat16((unsigned short)(key & 0x8000u ? key & 0x7fffu : ~key)));
}

template <typename T> __device__ __forceinline__ void load_vec(const T* p, float* v);
template <> __device__ __forceinline__ void load_vec<float>(const float* p, float* v) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
template <> __device__ __forceinline__ void load_vec<__nv_bfloat16>(const __nv_bfloat16* p, float* v) { load8(p, *reinterpret_cast<float(*)[8]>(v)); }

template <typename T> __device__ __forceinline__ uint4 pack_vec(const float* v);
template <> __device__ __forceinline__ uint4 pack_vec<float>(const float* v) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 pack_vec<__nv_bfloat16>(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// the largest of the numbers among 16 bytes at a time; NaN is none
template <typename T> struct RunMax;
template <> struct RunMax<float> {
  float m = -INFINITY;
  __device__ __forceinline__ void add(const uint4& v) {
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
  }
  __device__ __forceinline__ float get() const { return m; }
};
template <> struct RunMax<__nv_bfloat16> {
  __nv_bfloat162 m = __floats2bfloat162_rn(-INFINITY, -INFINITY);
  __device__ __forceinline__ static __nv_bfloat162 two(unsigned v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
  __device__ __forceinline__ void add(const uint4& v) { m = __hmax2(m, __hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w)))); }
  __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// 2^(d c) for -1000 < d c <= 0: table of 2^(i / 32) and the Taylor polynomial of degree 4 for the rest |r| <= 1/64 (Tang, 1989); 1.2e-12 of the value. The
// table lies in shared memory 16 times over, a copy for each lane of a half warp, so that a warp's loads meet no conflicts.
__device__ __forceinline__ double exp2_table(double d, double c, const double* table) {
  constexpr double BIG = 6755399441055744.0 / 32;         // 1.5 * 2^52 / 32: the sum's last bits count 32nds
  const double s = fma(d, c, BIG);
  const int n = __double2loint(s);
  const double r = fma(d, c, BIG - s);
  constexpr double L = 0.693147180559945309417;
  double p = fma(r, L * L * L * L / 24, L * L * L / 6);
  p = fma(p, r, L * L / 2);
  p = fma(p, r, L);
  const double t = table[(n & 31) * SM_COPIES];
  p = fma(p * r, t, t);
  return __hiloint2double(__double2hiint(p) + ((n >> 5) << 20), __double2loint(p));
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

// a float as a double by moving its fields: a conversion takes four times as long as a sum. Zero becomes 6e-39, infinity 2^128.
__device__ __forceinline__ int widen_high(float x) { return (int)(((unsigned)(__float_as_int(x) >> 3) & 0x8fffffffu) + 0x38000000u); }
// BF16 values have nothing in the lower word
template <typename T> __device__ __forceinline__ double widen(float x) { return __hiloint2double(widen_high(x), sizeof(T) == 2 ? 0 : (int)(__float_as_uint(x) << 29)); }
__device__ __forceinline__ float ex2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// A row as a CTA sees it: weights and bins of its logits. The largest logit is finite (rows with +inf are rewritten first).
template <typename T> struct SampleRow {
  float top;                            // the largest logit
  double c, wide_top;                   // log2(e) / T
  float half_top, ch, bins;             // half the largest logit; twice c, rounded; bins per two units of logit
  const double* table;
  float far;                            // least logit that weighs anything
  __device__ __forceinline__ double weight(float l) const { return l >= far ? exp2_table(widen<T>(l) - wide_top, c, table) : 0.0; }
  // half of what the largest logit is above l: a whole difference may be infinite, and infinity has no place in bins, nor octaves where c is zero
  __device__ __forceinline__ float half_down(float l) const { return fmaf(l, -0.5f, half_top); }
  // octaves of a logit against the largest
  __device__ __forceinline__ float octaves(float l) const { return half_down(l) * -ch; }
  // never falls as l does: a difference and a product with a factor that is not negative, each rounded, are monotone
  __device__ __forceinline__ float place(float l) const { return half_down(l) * bins; }
  __device__ __forceinline__ int bin(float l) const {
    const float x = place(l);
    return x < (float)(SM_BINS - 1) ? (int)x : SM_BINS - 1;
  }
};

// Sum over the block's threads in front of this one; `all`: over all of them. Every thread calls.
__device__ __forceinline__ double block_scan(double v, SampleShared& sh, int warp, int lane, double& all) {
  const double in = warp_scan64(v, lane);
  __syncthreads();
  if (lane == 31) sh.scan_mass[warp] = in;
  __syncthreads();
  double before = in - v;
  all = 0.0;
#pragma unroll
  for (int w = 0; w < SM_WARPS; ++w) { const double m = sh.scan_mass[w]; if (w < warp) before += m; all += m; }
  return before;
}

// list[0 .. n) in descending order, entries distinct, their lower halves within `span` from `base` on. Few entries count the larger ones, several threads per
// entry; more are placed by bins of both halves first, so that ties of one key spread over them, and count within their bin (a bitonic sort in
// shared memory took 5.5 us for 458 entries and 8.5 for 750, this 1.5 and 3.5).
__device__ __forceinline__ void sort_list(SampleShared& sh, int n, unsigned span, unsigned base, int tid, int warp, int lane) {
  if (n <= SM_SMALL) {
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    const int per = min(SM_THREADS / n2, 32), i = tid / per, at = tid % per;
    const unsigned long long me = i < n ? sh.list[i] : 0;
    int place = 0;
    if (i < n) for (int j = at; j < n; j += per) place += sh.list[j] > me;
    for (int o = per >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    __syncthreads();
    if (i < n && at == 0) sh.list[place] = me;
    __syncthreads();
    return;
  }
  constexpr int PER = SM_LIST / SM_THREADS, BINS = SM_LIST;
  unsigned long long me[PER];
  unsigned low = 0xffffffffu, high = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int i = tid + q * SM_THREADS;
    me[q] = i < n ? sh.list[i] : 0;
    if (i < n) { low = min(low, (unsigned)(me[q] >> 32)); high = max(high, (unsigned)(me[q] >> 32)); }
    sh.place[i] = 0;
  }
  if (tid == 0) { sh.reduce[0] = 0xffffffffu; sh.reduce[1] = 0; }
  __syncthreads();
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) { atomicMin(&sh.reduce[0], low); atomicMax(&sh.reduce[1], high); }
  __syncthreads();
  // distances from the end of the highest key's range: whole numbers below 2^32 * 2^31
  const unsigned lowest = sh.reduce[0];
  const unsigned long long top = ((unsigned long long)(sh.reduce[1] - lowest) + 1) * span;
  const float scale = (float)(BINS - 1) / (float)top;
  int bin[PER];
  unsigned slot[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    bin[q] = 0;
    if (tid + q * SM_THREADS < n) {
      const unsigned long long at = (unsigned long long)((unsigned)(me[q] >> 32) - lowest) * span + ((unsigned)me[q] - base);
      bin[q] = min((int)((float)(top - at) * scale), BINS - 1);
      slot[q] = atomicAdd(&sh.place[bin[q]], 1u);
    }
  }
  __syncthreads();
  unsigned c[PER], sum = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) { c[q] = sh.place[tid * PER + q]; sum += c[q]; }
  const unsigned upto = warp_scan_u32(sum, lane);
  if (lane == 31) sh.scan_count[warp] = upto;
  __syncthreads();
  unsigned at = upto - sum;
  for (int w = 0; w < warp; ++w) at += sh.scan_count[w];
#pragma unroll
  for (int q = 0; q < PER; ++q) { sh.place[tid * PER + q] = at; at += c[q]; }
  if (tid == 0) sh.place[BINS] = n;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (tid + q * SM_THREADS < n) sh.list[sh.place[bin[q]] + slot[q]] = me[q];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (tid + q * SM_THREADS < n) {
      const unsigned first = sh.place[bin[q]], last = sh.place[bin[q] + 1];
      slot[q] = first;
      for (unsigned j = first; j < last; ++j) slot[q] += sh.list[j] > me[q];
    }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (tid + q * SM_THREADS < n) sh.list[slot[q]] = me[q];
  __syncthreads();
}

// The list's n tokens (n <= SM_LIST) in the order's order, with their weights; then the first of them at which the prefix ends: `above` tokens of mass
// `mass_above` stand in front of the list. Returns how many of the list are kept, and their mass with mass_above in sh.total.
template <typename T>
__device__ __forceinline__ int find_border(SampleShared& sh, const SampleRow<T>& r, int n, unsigned above, double mass_above, bool use_k, int k, bool use_p, double target,
                                           int V, int tid, int warp, int lane) {
  if (tid == 0) sh.at = n - 1;
  __syncthreads();
  sort_list(sh, n, (unsigned)V, ~(unsigned)(V - 1), tid, warp, lane);
  const int per = (n + SM_THREADS - 1) / SM_THREADS, first = min(n, tid * per), last = min(n, first + per);
  double mine = 0.0;
  for (int i = first; i < last; ++i) { const double w = r.weight(logit_of<T>((unsigned)(sh.list[i] >> 32))); sh.w[i] = w; mine += w; }
  double all;
  double m = mass_above + block_scan(mine, sh, warp, lane, all);
  const double from = m;
  for (int i = first; i < last; ++i) {
    m += sh.w[i];
    if ((use_k && above + i + 1 >= (unsigned)k) || (use_p && m >= target)) { atomicMin(&sh.at, i); break; }
  }
  __syncthreads();
  const int at = sh.at;
  if (at >= first && at < last) {
    m = from;
    for (int i = first; i <= at; ++i) m += sh.w[i];
    sh.total = m;
  }
  __syncthreads();
  return at + 1;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 2)
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
  // 64-bit functions are hundreds of instructions that every warp would repeat: one warp calls each (256 rows of 151936: 105 -> 103 us)
  if (warp == 0) {
    static_assert(SM_TABLE == 32, "a lane per entry");
    const double t = exp2(lane / (double)SM_TABLE);
    for (int j = 0; j < SM_COPIES; ++j) sh.table[lane * SM_COPIES + (lane + j) % SM_COPIES] = t;
  }
  if (tid == 0) sh.list_n = 0;
  pdl_wait();
  float temp = a.temperature[row];
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.f, floor_p = a.min_p != nullptr ? a.min_p[row] : 0.f;
  float u = a.uniforms[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  // min-p as a distance of logits: rounded up below, so that for 32-bit logits the comparison is the one with the unrounded value
  const bool use_m = floor_p > 0.f && temp < INFINITY;
  if (warp == 1 && temp > 0.f) {
    const double c = 1.4426950408889634074 / (double)temp, below = use_m ? (double)temp * log((double)fminf(floor_p, 1.f)) : 0.0;
    if (lane == 0) { sh.c = c; sh.below = below; }
  }
  auto answer = [&](int id, float prob) { a.ids[row] = id; if (a.probs != nullptr) a.probs[row] = prob; };

  // ---- 1: logits into shared memory, their largest. Four loads of a thread are on their way at a time. NaN stays: no comparison lets it through ----
  RunMax<T> run_max;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  for (int i0 = lane * VEC; i0 < a.seg; i0 += 4 * STEP) {
    uint4 v[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int i = i0 + g * STEP, at = warp * a.seg + i;
      if (i < a.seg && vec && at + VEC <= have) {
        v[g] = *reinterpret_cast<const uint4*>(src + at);
      } else {
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = i < a.seg && at + e < have ? to_float(src[at + e]) : -INFINITY;
        v[g] = pack_vec<T>(f);
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int i = i0 + g * STEP;
      if (i >= a.seg) break;
      run_max.add(v[g]);
      *reinterpret_cast<uint4*>(mine + i) = v[g];
    }
  }
  float mine_top = run_max.get();                        // of this thread's tokens
  {
    const float m = warp_max(mine_top);
    if (lane == 0) sh.warp_top[warp] = m;
  }
  __syncwarp();
  cluster_wait();
  __syncthreads();
  if (tid < C) {
    float m = sh.warp_top[0];
    for (int w = 1; w < SM_WARPS; ++w) m = fmaxf(m, sh.warp_top[w]);
    push_u32(&sh.top[rank], tid, __float_as_uint(m));
  }
  cluster_sync_all();
  SampleRow<T> r;
  r.table = sh.table + lane % SM_COPIES;
  r.top = sh.top[0];
  for (int i = 1; i < C; ++i) r.top = fmaxf(r.top, sh.top[i]);
  const bool greedy = !(temp > 0.f);
  if (greedy || r.top == -INFINITY) {
    // the lowest id of the largest logit
    unsigned best = 0xffffffffu;
    if (mine_top == r.top)
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
      answer(none ? 0 : (int)best, none ? 0.f : 1.f);
    }
    return;
  }
  if (r.top == INFINITY) {
    // +inf stands for equal finite logits above all others'
    for (int i = lane * VEC; i < a.seg; i += STEP)
#pragma unroll
      for (int e = 0; e < VEC; ++e) from_float(mine + i + e, to_float(mine[i + e]) == INFINITY ? 0.f : -INFINITY);
    mine_top = mine_top == INFINITY ? 0.f : -INFINITY;
    r.top = 0.f;
  }
  double below = sh.below;
  r.c = sh.c;
  if (temp < 0x1p-80f && fabsf(r.top) < 0x1p-40f) {
    // Logits and temperature times 2^90 draw as before, and then no zero and no subnormal logit is nearer to the largest than widen() tells apart; what this takes to
    // -inf weighs nothing. Above 2^-40 numbers lie 2^-64 and more apart, so that at these temperatures only the largest logit weighs anything.
    constexpr float UP = 0x1p90f;
    for (int i = lane * VEC; i < a.seg; i += STEP)
#pragma unroll
      for (int e = 0; e < VEC; ++e) from_float(mine + i + e, to_float(mine[i + e]) * UP);
    mine_top *= UP; r.top *= UP; temp *= UP;
    r.c *= 1.0 / UP; below *= UP;
  }
  r.wide_top = widen<T>(r.top);
  r.half_top = 0.5f * r.top;
  r.ch = fminf((float)(r.c * 2.0), 2e30f);
  r.bins = fminf((float)(r.c * 32.0), 2e30f);
  const bool use_k = k > 0 && k < a.V, use_p = p < 1.f;
  r.far = fmaxf(r.ch > 0.f ? __fadd_ru(r.top, 2.f * SM_FAR / r.ch) : -INFINITY, -3.4028235e38f);      // rounded up: the next number below may lie thousands of octaves lower
  const float least = use_m ? fminf(r.top, __double2float_ru((double)r.top + below)) : -INFINITY;

  // The draw within the run of ids of warp `owner` of this CTA, by all of its warps: the lowest id at which the sum of kept weights, `from` in front of
  // the run, passes the goal. Shared memory holds runs of 24 steps at most; their sums first, then the step's tokens (48 rows of 128256 7 us
  // less than with one warp that walks step by step).
  auto walk = [&](int owner, double from, double goal, unsigned border_key, int border_id, double kept_all) {
    const T* run = slice + owner * a.seg;
    const int run_id = first + owner * a.seg, steps = a.seg / STEP;
    auto weigh = [&](int step, double (&w)[VEC]) {
      const int i = step * STEP + lane * VEC;
      float v[VEC];
      load_vec<T>(run + i, v);
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const unsigned key = key_of<T>(v[e]);
        const bool kept = v[e] >= least && (key > border_key || (key == border_key && run_id + i + e <= border_id));
        w[e] = kept ? r.weight(v[e]) : 0.0;
        sum += w[e];
      }
      return sum;
    };
    double w[VEC];
    for (int step = warp; step < steps; step += SM_WARPS) {
      const double sum = warp_sum64(weigh(step, w));
      if (lane == 0) sh.step_sum[step] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    const double mine_sum = lane < steps ? sh.step_sum[lane] : 0.0, upto_step = warp_scan64(mine_sum, lane);
    // the first step that passes, or the last one of any mass, as for tokens below
    const unsigned ends = __ballot_sync(0xffffffffu, mine_sum > 0.0 && from + upto_step > goal);
    const unsigned any_step = __ballot_sync(0xffffffffu, mine_sum > 0.0);
    const int step = ends ? __ffs(ends) - 1 : 31 - __clz(any_step);
    const double before = from + __shfl_sync(0xffffffffu, upto_step - mine_sum, step);
    const double sum = weigh(step, w);
    const double upto = warp_scan64(sum, lane);
    double x = before + (upto - sum);
    int got = -1, some = -1;
    double got_w = 0.0, some_w = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      x += w[e];
      if (w[e] > 0.0) {
        some = run_id + step * STEP + lane * VEC + e; some_w = w[e];
        if (got < 0 && x > goal) { got = some; got_w = w[e]; }
      }
    }
    // the first that passes; the sums' last bits may leave the goal behind the last token
    const unsigned vote = __ballot_sync(0xffffffffu, got >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
    if (vote ? lane == __ffs(vote) - 1 : lane == 31 - __clz(any)) answer(vote ? got : some, (float)((vote ? got_w : some_w) / kept_all));
  };

  // ---- 2: the mass, and a logit that k tokens reach ----
  float my_cut = INFINITY;
  if (use_k) {
    const int k_here = (int)(((long long)k * have + a.V - 1) / a.V);          // in proportion to the slice: k in all, or more
    if (k_here > 0) {
      // Of the threads' largest logits, by bins of 1/4 octave: those down to the bin in which the k_here-th lies are k_here at least.
      if (tid < 256) sh.count[tid] = 0;
      if (tid == 0) { sh.at = -1; sh.reduce[0] = 0xffffffffu; }
      __syncthreads();
      const int b = mine_top > -INFINITY ? min(r.bin(mine_top) >> 2, 255) : 256;
      if (b < 256) atomicAdd(&sh.count[b], 1u);
      __syncthreads();
      if (warp == 0) {
        unsigned c[8], sum = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) { c[q] = sh.count[lane * 8 + q]; sum += c[q]; }
        unsigned at = warp_scan_u32(sum, lane) - sum;
#pragma unroll
        for (int q = 0; q < 8; ++q) { if (at < (unsigned)k_here && at + c[q] >= (unsigned)k_here) sh.at = lane * 8 + q; at += c[q]; }
      }
      __syncthreads();
      const unsigned key = __reduce_min_sync(0xffffffffu, b <= sh.at ? order_key(mine_top) : 0xffffffffu);
      if (lane == 0) atomicMin(&sh.reduce[0], key);
      __syncthreads();
      my_cut = sh.at < 0 ? -INFINITY : logit_of<float>(sh.reduce[0]);
    }
  }
  if (use_p || !use_k) {
    // the draw's mass is that of the kept tokens
    double s = 0.0;
    const float from = fmaxf(use_p ? -INFINITY : least, r.far);
    if (mine_top >= from)
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          // what lies below gives some number or other, which is not added
          const double w = exp2_table(widen<T>(v[e]) - r.wide_top, r.c, r.table);
          s = v[e] >= from ? s + w : s;
        }
      }
    s = warp_sum64(s);
    if (lane == 0) sh.warp_sum[warp] = s;
  }
  __syncthreads();
  if (tid < C) {
    double s = 0.0;
    if (use_p || !use_k) for (int w = 0; w < SM_WARPS; ++w) s += sh.warp_sum[w];
    push_f64(&sh.mass[rank], tid, s);
    push_u32(&sh.cut[rank], tid, __float_as_uint(my_cut));
  }
  cluster_sync_all();
  double s = 0.0;
  float k_cut = INFINITY;
  for (int i = 0; i < C; ++i) { s += sh.mass[i]; k_cut = fminf(k_cut, sh.cut[i]); }

  // kept: key > border_key, or equal and id <= border_id; of those only logits >= least
  unsigned border_key = 0;
  int border_id = 0x7fffffff;
  double kept_all = s;                                   // mass of all kept tokens
  if (use_k || use_p) {
    // ---- 3: candidates ----
    const double target = use_p ? fmax((double)p, 0.0) * s : 0.0;
    float cut = fmaxf(least, use_k ? k_cut : -INFINITY);
    if (use_p) {
      // borders lie at weights of (1 - P) S / V and more; a thousandth is left for the roundings
      if (warp == 0) {
        const double away = log(0.999 * (1.0 - fmax((double)p, 0.0)) * s / a.V) * (double)temp;
        if (lane == 0) sh.below = away;
      }
      __syncthreads();
      cut = fmaxf(cut, fminf(r.top, __double2float_rd((double)r.top + sh.below)));
    }
    const bool some = mine_top >= cut && mine_top > -INFINITY;
    // 16 bytes of which none is a candidate are seen by their largest
    auto none_in = [&](int i) { RunMax<T> chunk; chunk.add(*reinterpret_cast<const uint4*>(mine + i)); return !(chunk.get() >= cut); };
    int n = 0;
    if (some)
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        if (none_in(i)) continue;
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) n += v[e] >= cut && v[e] > -INFINITY;
      }
    const int in_warp = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh.scan_count[warp] = in_warp;
    __syncthreads();
    const int in_cta = __reduce_add_sync(0xffffffffu, lane < SM_WARPS ? sh.scan_count[lane] : 0u);
    // a CTA with more than its part of the list leaves the row to the general path
    const int share = SM_LIST / C;
    if (tid < C) push_u32(&sh.candidates[rank], tid, in_cta);
    if (in_cta <= share && n > 0) {
      const unsigned slot0 = push_take(&sh.list_n, 0, n);          // at most SM_LIST in all
      unsigned slot = slot0;
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        if (none_in(i)) continue;
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (v[e] >= cut && v[e] > -INFINITY) push_u64(&sh.list[slot++], 0, (unsigned long long)key_of<T>(v[e]) << 32 | (unsigned)~(id0 + i + e));
      }
    }
    cluster_sync_all();
    int all = 0, most = 0;
    for (int i = 0; i < C; ++i) { all += sh.candidates[i]; most = max(most, sh.candidates[i]); }
    if (most <= share) {
      if (rank != 0) return;
      if (all <= 32) {
        // few candidates, what peaked distributions leave: one warp without a barrier, a token per lane
        if (warp != 0) return;
        const bool here = lane < all;
        const unsigned long long entry = here ? sh.list[lane] : 0;
        const double weight = here ? r.weight(logit_of<T>((unsigned)(entry >> 32))) : 0.0;
        int place = 0;
        for (int j = 0; j < all; ++j) place += sh.list[j] > entry;
        __syncwarp();
        if (here) { sh.list[place] = entry; sh.w[place] = weight; }
        __syncwarp();
        double w = here ? sh.w[lane] : 0.0;
        const double upto = warp_scan64(w, lane);
        const unsigned ends = __ballot_sync(0xffffffffu, here && ((use_k && lane + 1 >= k) || (use_p && upto >= target)));
        const int last_kept = ends ? __ffs(ends) - 1 : all - 1;
        const double total = __shfl_sync(0xffffffffu, upto, last_kept), goal = (double)u * total;
        // the kept ones by id
        const unsigned id = here ? ~(unsigned)sh.list[lane] : 0u;
        const bool kept = lane <= last_kept;
        place = 0;
        for (int j = 0; j <= last_kept; ++j) place += ~(unsigned)sh.list[j] < id;
        __syncwarp();
        if (kept) { sh.list[place] = id; sh.w[place] = w; }
        __syncwarp();
        w = kept ? sh.w[lane] : 0.0;
        const double m = warp_scan64(w, lane);
        const unsigned pass = __ballot_sync(0xffffffffu, w > 0.0 && m > goal), some_w = __ballot_sync(0xffffffffu, w > 0.0);
        if (lane == (pass ? __ffs(pass) - 1 : 31 - __clz(some_w))) answer((int)sh.list[lane], (float)(w / total));          // the sums' last bits may leave the goal behind the last token
        return;
      }
      const int kept = find_border<T>(sh, r, all, 0, 0.0, use_k, k, use_p, target, a.V, tid, warp, lane);
      const double goal = (double)u * sh.total;
      // the kept ones by id: ~id << 32 | place, descending
      const int per_thread = (kept + SM_THREADS - 1) / SM_THREADS;
      unsigned long long hold[SM_LIST / SM_THREADS];
#pragma unroll
      for (int q = 0; q < SM_LIST / SM_THREADS; ++q) {
        const int i = tid + q * SM_THREADS;
        hold[q] = i < kept ? (sh.list[i] << 32) | (unsigned)i : 0;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < SM_LIST / SM_THREADS; ++q) { const int i = tid + q * SM_THREADS; if (i < kept) sh.list[i] = hold[q]; }
      if (tid == 0) { sh.at = 0x7fffffff; sh.list_n = -1; }
      __syncthreads();
      sort_list(sh, kept, SM_LIST, 0u, tid, warp, lane);
      const int f0 = min(kept, tid * per_thread), f1 = min(kept, f0 + per_thread);
      double mass = 0.0, total;
      for (int i = f0; i < f1; ++i) mass += sh.w[(unsigned)sh.list[i]];
      double m = block_scan(mass, sh, warp, lane, total);
      int last = -1;
      for (int i = f0; i < f1; ++i) {
        const double w = sh.w[(unsigned)sh.list[i]];
        m += w;
        if (w > 0.0) { last = i; if (m > goal) { atomicMin(&sh.at, i); break; } }
      }
      if (last >= 0) atomicMax(&sh.list_n, last);
      __syncthreads();
      if (tid == 0) {
        const unsigned long long x = sh.list[sh.at == 0x7fffffff ? sh.list_n : sh.at];          // the sums' last bits may leave the goal behind the last token
        answer((int)~(unsigned)(x >> 32), (float)(sh.w[(unsigned)x] / sh.total));
      }
      return;
    }
    // ---- 4: the general path ----
    // the bins divide the range of the candidates, where it is known
    if (cut > -INFINITY && r.half_down(cut) > 0.f) r.bins = fminf(r.bins * 64.f, (float)(SM_BINS - 1) / r.half_down(cut));
    const float per_bin = r.bins > 0.f ? r.ch / r.bins : 0.f;
    __syncthreads();
    for (int i = tid; i < SM_BINS; i += SM_THREADS) { sh.all_count[i] = 0; sh.all_high[i] = 0; sh.all_low[i] = 0; sh.count[i] = 0; sh.mass_of[i] = 0; }
    if (tid == 0) sh.list_n = 0;
    cluster_sync_all();                                  // CTA 0's sums are clear, the lists forgotten
    if (some)
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (!(v[e] >= cut) || v[e] == -INFINITY) continue;
          const int b = r.bin(v[e]);
          if (use_p) {
            // in units of 2^-14 of the power of two above the bin's weights; 120 octaves and more below the largest weigh nothing
            const float x = r.octaves(v[e]), up = floorf((float)b * per_bin);
            if (up < 120.f) atomicAdd(&sh.mass_of[b], (unsigned)__float2int_rn(ex2_approx(x + up) * 16384.f));
          }
          atomicAdd(&sh.count[b], 1u);
        }
      }
    __syncthreads();
    for (int i = tid; i < SM_BINS; i += SM_THREADS)
      if (sh.count[i]) {
        push_add(&sh.all_count[i], 0, sh.count[i]);
        if (use_p) { push_add(&sh.all_high[i], 0, sh.mass_of[i] >> 16); push_add(&sh.all_low[i], 0, sh.mass_of[i] & 0xffffu); }
      }
    cluster_sync_all();
    if (rank == 0) {
      constexpr int PER = SM_BINS / SM_THREADS;
      unsigned c[PER], c_sum = 0;
      double m[PER], m_sum = 0.0;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int b = tid * PER + q;
        const float up = floorf((float)b * per_bin);
        c[q] = sh.all_count[b];
        m[q] = use_p && up < 120.f ? ((double)sh.all_high[b] * 65536.0 + (double)sh.all_low[b]) * power_of_2(-14 - (int)up) : 0.0;
        c_sum += c[q]; m_sum += m[q];
        sh.all_count[b] = 0; sh.all_high[b] = 0; sh.all_low[b] = 0;
      }
      const unsigned c_in = warp_scan_u32(c_sum, lane);
      if (lane == 31) sh.scan_count[warp] = c_in;
      if (tid == 0) sh.found = SampleFound{SM_BINS, 0, 0, 0};
      double m_all;
      double m_at = block_scan(m_sum, sh, warp, lane, m_all);
      unsigned c_at = c_in - c_sum;
      for (int w = 0; w < warp; ++w) c_at += sh.scan_count[w];
      // The masses are within 1e-4 of themselves: in the first bin behind which the target may be reached, or in a later one up to the first behind which
      // it surely is, lies the border.
      const double lo_target = target * (1.0 - 1e-4), hi_target = target * (1.0 + 1e-4);
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const unsigned c_to = c_at + c[q];
        const double m_to = m_at + m[q];
        if (c[q]) {
          const bool maybe = (use_k && c_to >= (unsigned)k) || (use_p && m_to >= lo_target), before = (use_k && c_at >= (unsigned)k) || (use_p && c_at > 0 && m_at >= lo_target);
          const bool sure = (use_k && c_to >= (unsigned)k) || (use_p && m_to >= hi_target), sure_before = (use_k && c_at >= (unsigned)k) || (use_p && c_at > 0 && m_at >= hi_target);
          if (maybe && !before) atomicMin(&sh.found.lo, tid * PER + q);
          if (!sure_before && (sure || maybe)) atomicMax(&sh.found.hi, tid * PER + q);
        }
        c_at = c_to; m_at = m_to;
      }
      __syncthreads();
      const int lo = sh.found.lo, hi = sh.found.hi;
#pragma unroll
      for (int q = PER - 1; q >= 0; --q) {
        const int b = tid * PER + q;
        c_at -= c[q];
        if (b >= lo && b <= hi && c[q]) atomicAdd(&sh.found.count, (int)c[q]);
        if (b == lo) sh.found.above = c_at;
      }
      __syncthreads();
      if (tid > 0 && tid < C) {
        push_u32(&sh.found.lo, tid, (unsigned)lo); push_u32(&sh.found.hi, tid, (unsigned)hi); push_u32(&sh.found.count, tid, (unsigned)sh.found.count);
        push_u32(&sh.found.above, tid, sh.found.above);
      }
    }
    cluster_sync_all();
    // the border's bins; none: all candidates are kept, and lie in front of bin SM_BINS
    const int lo = sh.found.lo, hi = sh.found.hi;
    unsigned above = lo < SM_BINS ? sh.found.above : 0u;
    unsigned key_lo = 0, key_hi = 0xffffffffu;
    int left = lo < SM_BINS ? sh.found.count : 0;
    bool ties = false;
    // bins of too many tokens: their keys are divided by count alone, down to the key up to which k or the list's length lead; masses are met in FP64 below
    auto inside = [&](float l, unsigned key) { const int b = r.bin(l); return l >= cut && l > -INFINITY && b >= lo && b <= hi && key >= key_lo && key <= key_hi; };
    double mass_above = 0.0;
    while (left > SM_LIST) {
      unsigned kmin = 0xffffffffu, kmax = 0;
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const unsigned key = key_of<T>(v[e]);
          if (inside(v[e], key)) { kmin = min(kmin, key); kmax = max(kmax, key); }
        }
      }
      kmin = __reduce_min_sync(0xffffffffu, kmin);
      kmax = __reduce_max_sync(0xffffffffu, kmax);
      __syncthreads();
      if (tid == 0) { sh.reduce[0] = 0xffffffffu; sh.reduce[1] = 0; }
      __syncthreads();
      if (lane == 0) { atomicMin(&sh.reduce[0], kmin); atomicMax(&sh.reduce[1], kmax); }
      __syncthreads();
      if (tid < C) { push_u32(&sh.key_min[rank], tid, sh.reduce[0]); push_u32(&sh.key_max[rank], tid, sh.reduce[1]); }
      cluster_sync_all();
      key_lo = sh.key_min[0]; key_hi = sh.key_max[0];
      for (int i = 1; i < C; ++i) { key_lo = min(key_lo, sh.key_min[i]); key_hi = max(key_hi, sh.key_max[i]); }
      if (key_lo == key_hi) { ties = true; break; }
      // the upper half of the keys: how many, and what mass with all in front of them
      const unsigned mid = key_lo + (key_hi - key_lo + 1) / 2;
      unsigned n_up = 0;
      double m = 0.0;
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const unsigned key = key_of<T>(v[e]);
          const bool in = inside(v[e], key);
          n_up += in && key >= mid;
          const int b = r.bin(v[e]);
          if (use_p && v[e] >= cut && v[e] > -INFINITY && (b < lo || (b <= hi && key >= mid))) m += r.weight(v[e]);
        }
      }
      n_up = __reduce_add_sync(0xffffffffu, n_up);
      m = warp_sum64(m);
      if (lane == 0) { sh.warp_ties[warp] = n_up; sh.warp_sum[warp] = m; }
      __syncthreads();
      if (tid < C) {
        double t = 0.0;
        unsigned c = 0;
        for (int w = 0; w < SM_WARPS; ++w) { t += sh.warp_sum[w]; c += sh.warp_ties[w]; }
        push_f64(&sh.mass[rank], tid, t);
        push_u32(&sh.ties[rank], tid, c);
      }
      cluster_sync_all();
      double upper = 0.0;
      int n_upper = 0;
      for (int i = 0; i < C; ++i) { upper += sh.mass[i]; n_upper += (int)sh.ties[i]; }
      // the border lies in the upper half if it is reached there
      if ((use_k && above + n_upper >= (unsigned)k) || (use_p && n_upper > 0 && upper >= target)) { key_lo = mid; left = n_upper; }
      else { key_hi = mid - 1; above += n_upper; left -= n_upper; }
    }
    // the mass in front of the border's bins (and keys) in FP64, warp by warp, without branches; the tokens among which the border lies into CTA 0's list
    double m = 0.0;
    unsigned n_ties = 0;
    // bins as numbers that r.bin rounds down: no number reaches the first one behind the last bin, nor NaN, which stands for it
    const float lo_x = lo < SM_BINS ? (float)lo : __uint_as_float(0x7fffffffu), hi_x = hi < SM_BINS - 1 ? (float)(hi + 1) : __uint_as_float(0x7fffffffu);
    const float cut_in = fmaxf(cut, -3.4028235e38f), heavy = fmaxf(cut_in, r.far);
    auto at_border = [&](float l) {
      const float x = r.place(l);
      const unsigned key = key_of<T>(l);
      return l >= cut_in && x >= lo_x && !(x >= hi_x) && key >= key_lo && key <= key_hi;
    };
    __syncthreads();                                     // the histogram's place is the list's
    if (some) {
      for (int i = lane * VEC; i < a.seg; i += STEP) {
        float v[VEC];
        load_vec<T>(mine + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float x = r.place(v[e]);
          const unsigned key = key_of<T>(v[e]);
          const bool until = !(x >= hi_x), front = !(x >= lo_x) || (until && key > key_hi), weighs = v[e] >= heavy;
          const double w = exp2_table(widen<T>(v[e]) - r.wide_top, r.c, r.table);
          m = weighs && front ? m + w : m;
          n_ties += v[e] >= cut_in && until && !front && key >= key_lo;
        }
      }
      if (n_ties > 0 && !ties) {
        unsigned slot = push_take(&sh.list_n, 0, n_ties);
        for (int i = lane * VEC; i < a.seg; i += STEP) {
          float v[VEC];
          load_vec<T>(mine + i, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (at_border(v[e])) push_u64(&sh.list[slot++], 0, (unsigned long long)key_of<T>(v[e]) << 32 | (unsigned)~(id0 + i + e));
        }
      }
    }
    m = warp_sum64(m);
    n_ties = __reduce_add_sync(0xffffffffu, n_ties);
    if (lane == 0) {
      sh.warp_sum[warp] = m; sh.warp_ties[warp] = n_ties;
      push_f64(&sh.part[rank * SM_WARPS + warp], 0, m);
    }
    __syncthreads();
    if (ties && tid < C) {
      // Counts and masses have places of their CTA's that the division by keys pushed to as well. Only after its end by ties has a barrier of the cluster passed
      // since they were read there; after its other end a peer may still be reading them.
      double t = 0.0;
      unsigned c = 0;
      for (int w = 0; w < SM_WARPS; ++w) { t += sh.warp_sum[w]; c += sh.warp_ties[w]; }
      push_u32(&sh.ties[rank], tid, c);
      push_f64(&sh.mass[rank], tid, t);
    }
    cluster_sync_all();
    if (ties) {
      // ---- ties of one key: as many of the lowest ids as are needed ----
      const double w_tie = r.weight(logit_of<T>(key_lo));
      unsigned all_ties = 0, before = 0;
      for (int i = 0; i < C; ++i) { if (i < rank) before += sh.ties[i]; all_ties += sh.ties[i]; mass_above += sh.mass[i]; }
      unsigned want = all_ties;
      if (use_k) want = min(want, (unsigned)k - above);
      if (use_p) {
        const double need = ceil((target - mass_above) / w_tie);
        if (need < (double)want) want = need < 1.0 ? 1u : (unsigned)need;
      }
      for (int w = 0; w < warp; ++w) before += sh.warp_ties[w];
      const unsigned taken = want <= before ? 0u : min(want - before, n_ties);
      if (lane == 0) push_f64(&sh.part[rank * SM_WARPS + warp], 0, m + (double)taken * w_tie);
      if (want > before && want <= before + n_ties) {    // this warp holds the last one
        unsigned at = before;
        for (int i = lane * VEC; i - lane * VEC < a.seg; i += STEP) {
          float v[VEC];
          unsigned here = 0;
          load_vec<T>(mine + i, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) here += inside(v[e], key_of<T>(v[e]));
          const unsigned upto = warp_scan_u32(here, lane);
          unsigned seen = at + upto - here;
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (inside(v[e], key_of<T>(v[e])) && ++seen == want) push_u32(&sh.border_id, 0, (unsigned)(id0 + i + e));
          at += __shfl_sync(0xffffffffu, upto, 31);
        }
      }
      cluster_sync_all();
    }
    if (rank == 0) {
      // the border, every warp's kept mass, and whose the draw is
      if (!ties && left > 0) {
        double front = 0.0;
        for (int i = tid; i < C * SM_WARPS; i += SM_THREADS) front += sh.part[i];
        block_scan(front, sh, warp, lane, mass_above);
        const int kept = find_border<T>(sh, r, left, above, mass_above, use_k, k, use_p, target, a.V, tid, warp, lane);
        if (tid < SM_PARTS) { sh.part_in[tid][0] = 0; sh.part_in[tid][1] = 0; sh.part_in[tid][2] = 0; }
        __syncthreads();
        for (int i = tid; i < kept; i += SM_THREADS) {
          // 2^50 and less; what weighs anything is at least a unit, so that its warp is seen to hold some
          const unsigned long long w = max((unsigned long long)(sh.w[i] * 1125899906842624.0), sh.w[i] > 0.0 ? 1ull : 0ull);
          unsigned* part = sh.part_in[(int)~(unsigned)sh.list[i] / a.seg];
          atomicAdd(part, (unsigned)(w >> 40)); atomicAdd(part + 1, (unsigned)(w >> 20) & 0xfffffu); atomicAdd(part + 2, (unsigned)w & 0xfffffu);
        }
        __syncthreads();
        if (tid < C * SM_WARPS) sh.part[tid] += (((double)sh.part_in[tid][0] * 1048576.0 + sh.part_in[tid][1]) * 1048576.0 + sh.part_in[tid][2]) * (1.0 / 1125899906842624.0);
        if (tid == 0) { sh.border_key = (unsigned)(sh.list[kept - 1] >> 32); sh.border_id = (int)~(unsigned)sh.list[kept - 1]; }
      } else if (tid == 0) {
        sh.border_key = ties ? key_lo : 0u;
        if (!ties) sh.border_id = 0x7fffffff;
      }
      __syncthreads();
      const double mine_part = tid < C * SM_WARPS ? sh.part[tid] : 0.0;
      double all_parts;
      const double from = block_scan(mine_part, sh, warp, lane, all_parts);
      const double goal = (double)u * all_parts;
      if (tid == 0) { sh.total = all_parts; sh.owner = SM_PARTS; sh.at = 0; }
      __syncthreads();
      // the first warp whose end passes the goal; the sums' last bits may leave it behind the last one
      if (mine_part > 0.0) { if (from + mine_part > goal) atomicMin(&sh.owner, tid); atomicMax(&sh.at, tid); }
      __syncthreads();
      const int owner = min(sh.owner, sh.at);
      if (tid == owner) sh.from = from;
      __syncthreads();
      if (tid > 0 && tid < C) {
        push_u32(&sh.owner, tid, (unsigned)owner); push_u32(&sh.border_key, tid, sh.border_key); push_u32(&sh.border_id, tid, (unsigned)sh.border_id);
        push_f64(&sh.from, tid, sh.from); push_f64(&sh.total, tid, sh.total);
      }
    }
    cluster_sync_all();
    border_key = sh.border_key; border_id = sh.border_id;
    kept_all = sh.total;
    if (sh.owner / SM_WARPS != rank) return;
    walk(sh.owner % SM_WARPS, sh.from, (double)u * kept_all, border_key, border_id, kept_all);
    return;
  }

  // ---- 3, without top-k and top-p: the draw from the warps' masses ----
  double before = 0.0, all = 0.0;
  int last = 0;                                          // the last CTA that holds any of the mass
  for (int i = 0; i < C; ++i) { if (i == rank) before = all; all += sh.mass[i]; if (sh.mass[i] > 0.0) last = i; }
  const double goal = (double)u * all, after = before + sh.mass[rank];
  if (!(goal >= before && (goal < after || rank == last) && sh.mass[rank] > 0.0)) return;
  // this CTA has it: the warp, then the token
  int owner = -1;
  double at = before, from = before;
  for (int w = 0; w < SM_WARPS; ++w) { if (sh.warp_sum[w] > 0.0 && (at <= goal || owner < 0)) { owner = w; from = at; } at += sh.warp_sum[w]; }
  walk(owner, from, goal, border_key, border_id, kept_all);
}

}  // namespace ff
using namespace ff;

template <typename T>
static int sample_launch(const SampleArgs& args, int rows, cudaStream_t stream) {
  constexpr int STEP = SM_STEP_BYTES / (int)sizeof(T), MOST = SM_MOST_SMEM;
  static_assert((MOST - (int)sizeof(SampleShared)) / (SM_WARPS * SM_STEP_BYTES) <= SM_MOST_STEPS, "a run's steps have a lane each");
  const int fixed = ((int)sizeof(SampleShared) + 15) / 16 * 16;
  SampleArgs a = args;
  // As many CTAs of at least 2048 tokens as stand on the GPU at once, two to an SM: a CTA has about 15 us of steps that wait, so a second wave costs more
  // than smaller CTAs save (64 rows of 128256, C = 8 in two waves / 4 in one: top-k, top-p and min-p together 37 / 29 us, top-p alone on flat rows 89 / 77; the other
  // way round only where few of the rows are flat, 46 / 57; 64 rows of 50257 with top-k 24 / 16). CTAs so large that an SM holds one are no gain where
  // rows wait anyway (256 rows of 128256, C = 4 / 2: 105 / 134).
  auto smem_of = [&](int n) { return (long long)((a.V + n * SM_WARPS - 1) / (n * SM_WARPS) + STEP) * SM_WARPS * sizeof(T) + fixed; };
  int c = SM_CLUSTER;
  while (c > 1 && smem_of(c / 2) <= MOST && (a.V < 2048 * c || (rows * c > 2 * sm_count() && 2 * (smem_of(c / 2) + 1024) <= 228 * 1024))) c /= 2;
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
