// Sampling one token per row of logits from given random numbers: temperature, top-k, min-p, top-p.
//
//   p_i = exp((z_i - max z) / t); kept: the k largest, of these p_i >= min_p, of these the shortest run in descending
//   order whose mass reaches top_p; token = the first kept i in vocabulary order with sum_{j <= i} p_j > u sum p.
//
// Which token comes out hangs on comparisons of long sums, so the masses are 64-bit fixed-point integers
// (round(p 2^46), fewer fraction bits for vocabularies above 2^16): sums are exact, the same in every order, and far finer than
// the gap between neighbouring tokens. p itself is computed in 64-bit floating point; a logit more than 33 t below the
// maximum has no mass and is never looked at again.
//
// One CTA per row. A histogram over z (bins of equal width below the maximum: monotone in z, and spread, where the
// bits of z would put most logits into a handful of bins) finds a cut below which nothing can be kept. If at most 1024
// logits lie above it - the usual settings - they are collected in shared memory, sorted, and everything else happens there: only these
// need the exponential. Otherwise the thresholds are narrowed down by further histograms over the bits of z, and the
// draw walks the vocabulary by halving it among the warps.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "serving.h"

namespace nc {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;      // candidates that are sorted in shared memory
constexpr float kReach = 33.0f;  // e^-33 < 2^-47: no mass beyond

// z as a number that orders like its bits: NaN becomes -infinity, -0 becomes 0.
__device__ __forceinline__ float clean(float z) { return z == z ? z + 0.0f : -CUDART_INF_F; }
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

template <class T>
struct RowView {
  const T* p;
  int n;
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 2) return clean(__bfloat162float(p[i]));
    else return clean(p[i]);
  }
  // f(index, z) for every element, by 16-byte loads between the first and the last aligned address
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int E = 16 / sizeof(T);
    const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int vecs = (n - head) / E;
    if (threadIdx.x < head) f(static_cast<int>(threadIdx.x), at(threadIdx.x));
#pragma unroll 2
    for (int v = threadIdx.x; v < vecs; v += kThreads) {
      const int i = head + v * E;
      const uint4 w = *reinterpret_cast<const uint4*>(p + i);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float z;
        if constexpr (sizeof(T) == 2) z = __uint_as_float((e & 1) ? (u[e / 2] & 0xffff0000u) : (u[e / 2] << 16));
        else z = __uint_as_float(u[e]);
        f(i + e, clean(z));
      }
    }
    for (int i = head + vecs * E + threadIdx.x; i < n; i += kThreads) f(i, at(i));
  }
};

// exp((z - zmax) / t) in 64 bits by argument reduction to |r| <= ln2 / 64 with a table of 2^(j/32) and the Taylor
// polynomial to the fifth power (remainder below 2^-47 of the value).
struct Exponent {
  double zmax, inv_t;
  const double* table;   // shared: 2^(j / 32)
  int fraction;          // bits behind the point of a mass
  float z_cut;           // below: no mass
  __device__ __forceinline__ double p(float z) const {
    const double x = (static_cast<double>(z) - zmax) * inv_t;
    constexpr double kPerLn2 = 46.16624130844682838;   // 32 / ln 2
    constexpr double kLn2Hi = 0x1.62e42fefa0000p-6, kLn2Lo = 0x1.cf79abc9e3b3ap-45;   // ln 2 / 32 in two parts
    const double kd = rint(x * kPerLn2);
    const int k = static_cast<int>(kd);
    const double r = fma(kd, -kLn2Lo, fma(kd, -kLn2Hi, x));
    const double q = r * fma(r, fma(r, fma(r, fma(r, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0);
    const double s = table[k & 31];
    return ldexp(fma(s, q, s), k >> 5);
  }
  __device__ __forceinline__ u64 mass_of(double p) const {   // round(p 2^fraction), p <= 1
    return static_cast<u64>(__double2ll_rn(p * static_cast<double>(1ull << fraction)));
  }
  __device__ __forceinline__ u64 mass(float z) const { return z < z_cut ? 0ull : z == static_cast<float>(zmax) ? 1ull << fraction : mass_of(p(z)); }
};

struct Shared {
  double table[32];
  u64 list[kList];             // sorted candidates: order key in the high half, ~index in the low
  u64 list_mass[kList];
  union {
    unsigned count[kBins];
    u64 mass[kBins];
  };
  u64 warp_sum[kWarps];
  float warp_max[kWarps], warp_min[kWarps];
  int warp_arg[kWarps];
  unsigned n;                  // candidates collected
  int bin;
  u64 below, inside;
  int lo, hi;
  u64 target;
  int answer;
};

__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Inclusive scan of one value per thread over the CTA; `total` of all.
__device__ __forceinline__ u64 block_scan(u64 v, Shared& sm, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) sm.warp_sum[warp] = v;
  __syncthreads();
  const u64 w = warp_scan(sm.warp_sum[lane], lane);
  total = __shfl_sync(0xffffffffu, w, 31);
  const u64 before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return v + (warp > 0 ? before : 0);
}

// Sorts n2 (a power of two) 64-bit values in shared memory, ascending or descending.
__device__ void sort_list(u64* v, int n2, bool descending) {
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n2 / 2; t += kThreads) {
        const int i = 2 * j * (t / j) + t % j, o = i + j;
        const u64 x = v[i], y = v[o];
        const bool up = ((i & k) == 0) != descending;
        if ((x > y) == up) v[i] = y, v[o] = x;
      }
    }
  __syncthreads();
}

// The first index at which the running weight (vocabulary order) exceeds `target`; w(i) is the weight of element i.
// The range is divided among the warps until one warp can walk it. `total` must exceed target.
template <class W>
__device__ int order_search(Shared& sm, int n, u64 target, W w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = n;
  while (hi - lo > 64) {
    const int seg = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int a = min(lo + warp * seg, hi), b = min(a + seg, hi);
    u64 s = 0;
    for (int i = a + lane; i < b; i += 32) s += w(i);
    s = warp_total(s);
    __syncthreads();
    if (lane == 0) sm.warp_sum[warp] = s;
    __syncthreads();
    if (warp == 0) {
      const u64 c = warp_scan(sm.warp_sum[lane], lane);
      const unsigned over = __ballot_sync(0xffffffffu, c > target);
      const int f = over ? __ffs(over) - 1 : kWarps - 1;
      if (lane == f) {
        sm.lo = min(lo + f * seg, hi), sm.hi = min(lo + (f + 1) * seg, hi);
        sm.target = target - (c - sm.warp_sum[lane]);
      }
    }
    __syncthreads();
    lo = sm.lo, hi = sm.hi, target = sm.target;
  }
  if (warp == 0) {
    int found = -1;
    u64 run = 0;
    for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
      const u64 x = i0 + lane < hi ? w(i0 + lane) : 0;
      const u64 c = warp_scan(x, lane) + run;
      const unsigned over = __ballot_sync(0xffffffffu, c > target);
      if (over) found = i0 + __ffs(over) - 1;
      run = __shfl_sync(0xffffffffu, c, 31);
    }
    if (lane == 0) sm.answer = found;
  }
  __syncthreads();
  const int r = sm.answer;
  __syncthreads();
  return r;
}

// Kept so far: elements with a key above `key`, and those equal to it up to index `last`.
struct Threshold {
  uint32_t key = 0;
  int last = 0x7fffffff;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

// Descending histogram search over the keys of the elements that `in` selects, all within [lo, hi]: the largest key at
// which the running weight (from the top) reaches `want` > 0. On return sm.below is the weight strictly above that key.
template <class T, class In, class W>
__device__ uint32_t key_search(Shared& sm, const RowView<T>& row, uint32_t lo, uint32_t hi, double want, u64 above, In in, W w) {
  while (lo < hi) {
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sm.mass[i] = 0;
    __syncthreads();
    row.each([&](int i, float z) {
      const uint32_t k = order_key(z);
      if (k >= lo && k <= hi && in(i, z, k)) atomicAdd(&sm.mass[(hi - k) >> shift], w(z));
    });
    __syncthreads();
    // two neighbouring bins per thread
    u64 total;
    const u64 x0 = sm.mass[2 * threadIdx.x], x1 = sm.mass[2 * threadIdx.x + 1];
    const u64 c1 = block_scan(x0 + x1, sm, total) + above, c0 = c1 - x1, before = c0 - x0;
    if (threadIdx.x == 0) sm.bin = -1;
    __syncthreads();
    const bool r0 = static_cast<double>(c0) >= want, rb = static_cast<double>(before) >= want, r1 = static_cast<double>(c1) >= want;
    if (r0 && !rb) sm.bin = 2 * threadIdx.x, sm.below = before;
    else if (r1 && !r0) sm.bin = 2 * threadIdx.x + 1, sm.below = c0;
    __syncthreads();
    int j = sm.bin;
    if (j < 0) {   // rounding of `want` past the total: the last key
      j = static_cast<int>((hi - lo) >> shift);
      if (threadIdx.x == 0) sm.below = above + total - sm.mass[j];
      __syncthreads();
    }
    above = sm.below;
    const uint32_t new_hi = hi - (static_cast<uint32_t>(j) << shift);
    const u64 span = (1ull << shift) - 1;
    lo = static_cast<u64>(new_hi) - lo > span ? static_cast<uint32_t>(new_hi - span) : lo;
    hi = new_hi;
    __syncthreads();
  }
  if (threadIdx.x == 0) sm.below = above;
  __syncthreads();
  return lo;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) sample_rows_kernel(const SampleArgs a) {
  __shared__ Shared sm;
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const RowView<T> row{static_cast<const T*>(a.logits) + r * a.ld, a.vocab};
  const float t = a.temperature_rows != nullptr ? a.temperature_rows[r] : a.temperature;
  const float top_p = a.top_p_rows != nullptr ? a.top_p_rows[r] : a.top_p;
  const float min_p = a.min_p_rows != nullptr ? a.min_p_rows[r] : a.min_p;
  int k = a.top_k_rows != nullptr ? a.top_k_rows[r] : a.top_k;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  if (threadIdx.x < 32) sm.table[threadIdx.x] = exp2(threadIdx.x / 32.0);

  // ---- the largest logit (lowest index of equals) and the smallest above -infinity
  float zmax = -CUDART_INF_F, zmin = CUDART_INF_F;
  int arg = 0x7fffffff;
  row.each([&](int i, float z) {
    if (z > zmax || (z == zmax && i < arg)) zmax = z, arg = i;
    if (z > -CUDART_INF_F) zmin = fminf(zmin, z);
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float oz = __shfl_xor_sync(0xffffffffu, zmax, o);
    const int oi = __shfl_xor_sync(0xffffffffu, arg, o);
    if (oz > zmax || (oz == zmax && oi < arg)) zmax = oz, arg = oi;
    zmin = fminf(zmin, __shfl_xor_sync(0xffffffffu, zmin, o));
  }
  if (lane == 0) sm.warp_max[warp] = zmax, sm.warp_arg[warp] = arg, sm.warp_min[warp] = zmin;
  __syncthreads();
  zmax = sm.warp_max[lane], arg = sm.warp_arg[lane], zmin = sm.warp_min[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float oz = __shfl_xor_sync(0xffffffffu, zmax, o);
    const int oi = __shfl_xor_sync(0xffffffffu, arg, o);
    if (oz > zmax || (oz == zmax && oi < arg)) zmax = oz, arg = oi;
    zmin = fminf(zmin, __shfl_xor_sync(0xffffffffu, zmin, o));
  }
  if (zmax == -CUDART_INF_F || !(t > 0.0f) || k == 1 || !(top_p > 0.0f) || !(min_p <= 1.0f)) {
    if (threadIdx.x == 0) a.out[r] = zmax == -CUDART_INF_F ? -1 : arg;
    return;
  }
  Exponent ex;
  ex.zmax = static_cast<double>(zmax), ex.inv_t = 1.0 / static_cast<double>(t), ex.table = sm.table;
  int log_v = 0;
  while ((1ll << log_v) < a.vocab) ++log_v;
  ex.fraction = min(46, 62 - log_v);
  ex.z_cut = fmaxf(zmax - kReach * t, -3.402823466e38f);   // -infinity has no mass at any temperature
  const double u = fmax(static_cast<double>(a.u[r]), 0.0), pmin = static_cast<double>(min_p), want_p = static_cast<double>(top_p);
  const bool nucleus = top_p < 1.0f, filtered = k < a.vocab || nucleus || min_p > 0.0f;
  const uint32_t max_key = order_key(zmax);

  Threshold cut;                    // what top-k and top-p keep, when the long way is taken
  cut.key = order_key(ex.z_cut), cut.last = 0x7fffffff;
  if (filtered) {
    const float width = fminf(zmax - zmin, kReach * t);
    const float per = width > 0.0f ? static_cast<float>(kBins) / width : 0.0f;
    auto bin_of = [&](float z) { return z == zmax ? 0 : min(static_cast<int>((zmax - z) * per), kBins - 1); };
    for (int i = threadIdx.x; i < kBins; i += kThreads) sm.count[i] = 0;
    if (threadIdx.x == 0) sm.bin = kBins - 1, sm.n = 0;
    __syncthreads();
    row.each([&](int, float z) {
      if (z >= ex.z_cut) atomicAdd(&sm.count[bin_of(z)], 1u);
    });
    __syncthreads();
    // the first bin at which k logits are reached, and the last one that min_p can keep anything of
    u64 total;
    const unsigned n0 = sm.count[2 * threadIdx.x], n1 = sm.count[2 * threadIdx.x + 1];
    const u64 c1 = block_scan(n0 + n1, sm, total), c0 = c1 - n1, before = c0 - n0;
    if (c0 >= static_cast<u64>(k) && before < static_cast<u64>(k)) sm.bin = 2 * threadIdx.x;
    else if (c1 >= static_cast<u64>(k) && c0 < static_cast<u64>(k)) sm.bin = 2 * threadIdx.x + 1;
    __syncthreads();
    const int bin_k = sm.bin;
    int bin_m = kBins - 1;
    if (min_p > 0.0f) {   // rounded down generously; the exact comparison follows
      const float z = zmax + t * logf(min_p) * 1.0001f - 1e-5f * (fabsf(zmax) + 1.0f);
      bin_m = z > ex.z_cut ? bin_of(z) : kBins - 1;
    }
    const int bin_cut = min(bin_k, bin_m);
    __syncthreads();
    if (bin_cut / 2 == static_cast<int>(threadIdx.x)) sm.inside = bin_cut & 1 ? c1 : c0;
    if (bin_k / 2 == static_cast<int>(threadIdx.x)) sm.below = bin_k & 1 ? c0 : before;
    __syncthreads();
    const u64 n_cut = sm.inside, above_k = sm.below;

    if (n_cut <= kList) {
      // ---- the short way: collect, sort, decide
      row.each([&](int i, float z) {
        if (z >= ex.z_cut && bin_of(z) <= bin_cut)
          sm.list[atomicAdd(&sm.n, 1u)] = (static_cast<u64>(order_key(z)) << 32) | static_cast<uint32_t>(~i);
      });
      __syncthreads();
      const int n = static_cast<int>(sm.n);
      int n2 = 2;
      while (n2 < n) n2 <<= 1;
      for (int i = n + threadIdx.x; i < n2; i += kThreads) sm.list[i] = 0;
      sort_list(sm.list, n2, true);
      const int i = threadIdx.x;
      u64 mine = 0, total_k;
      if (i < n && i < k) {
        const float z = key_value(static_cast<uint32_t>(sm.list[i] >> 32));
        const double p = z == zmax ? 1.0 : ex.p(z);
        if (i == 0 || p >= pmin) mine = ex.mass_of(p);
      }
      const u64 incl = block_scan(mine, sm, total_k);
      bool keep = i < n && i < k && mine > 0;
      if (nucleus && i > 0) keep = keep && static_cast<double>(incl - mine) < want_p * static_cast<double>(total_k);
      // Back to vocabulary order: index in the high half, place in the list in the low; what is not kept goes last.
      sm.list_mass[i] = keep ? mine : 0;
      const uint32_t index = i < n ? ~static_cast<uint32_t>(sm.list[i]) : 0xffffffffu;
      __syncthreads();
      if (i < n2) sm.list[i] = (static_cast<u64>(keep ? index : 0xffffffffu) << 32) | static_cast<uint32_t>(i);
      sort_list(sm.list, n2, false);
      u64 w = i < n2 && (sm.list[i] >> 32) != 0xffffffffu ? sm.list_mass[static_cast<uint32_t>(sm.list[i])] : 0;
      u64 kept;
      const u64 cum = block_scan(w, sm, kept);
      const u64 target = static_cast<u64>(u * static_cast<double>(kept));
      const u64 goal = target < kept ? target : kept - 1;
      if (w > 0 && cum > goal && cum - w <= goal) a.out[r] = static_cast<long long>(sm.list[i] >> 32);
      return;
    }

    // ---- the long way: thresholds by narrowing histograms
    auto passes_min_p = [&](float z) { return min_p <= 0.0f || z == zmax || ex.p(z) >= pmin; };
    if (above_k < static_cast<u64>(k) && total > static_cast<u64>(k)) {
      auto in_bin = [&](int, float z, uint32_t) { return z >= ex.z_cut && bin_of(z) == bin_k; };
      const uint32_t key = key_search(sm, row, order_key(ex.z_cut), max_key, static_cast<double>(k), above_k, in_bin,
                                      [](float) { return 1ull; });
      const u64 ties = static_cast<u64>(k) - sm.below;   // that many of the equals are kept
      __syncthreads();
      cut.key = key;
      cut.last = order_search(sm, a.vocab, ties - 1, [&](int i) { return order_key(row.at(i)) == key ? 1ull : 0ull; });
      if (cut.last < 0) cut.last = 0x7fffffff;
    }
    if (nucleus) {
      const Threshold top = cut;
      auto in = [&](int i, float z, uint32_t key) { return top.keeps(key, i) && z >= ex.z_cut && passes_min_p(z); };
      u64 mass = 0, all;
      row.each([&](int i, float z) {
        if (in(i, z, order_key(z))) mass += ex.mass(z);
      });
      block_scan(mass, sm, all);
      const double want = want_p * static_cast<double>(all);
      const uint32_t key = key_search(sm, row, order_key(ex.z_cut), max_key, want, 0ull, in, [&](float z) { return ex.mass(z); });
      const u64 above = sm.below, each = ex.mass(key_value(key));
      __syncthreads();
      // equals are kept while the mass before them is short of `want`
      double need = each > 0 ? ceil((want - static_cast<double>(above)) / static_cast<double>(each)) : 1.0;
      u64 ties = need < 1.0 ? 1 : static_cast<u64>(need);
      while (ties > 1 && static_cast<double>(above + (ties - 1) * each) >= want) --ties;
      while (static_cast<double>(above + ties * each) < want && ties < static_cast<u64>(a.vocab)) ++ties;
      const int last = order_search(sm, a.vocab, ties - 1, [&](int i) {
        const float z = row.at(i);
        return order_key(z) == key && top.keeps(key, i) ? 1ull : 0ull;
      });
      cut.key = key;
      if (key != top.key || last >= 0) cut.last = last < 0 ? 0x7fffffff : last;
    }
  }

  // ---- the draw, over the vocabulary
  auto weight = [&](int i) {
    const float z = row.at(i);
    if (z < ex.z_cut || !cut.keeps(order_key(z), i)) return 0ull;
    if (z == zmax) return 1ull << ex.fraction;
    const double p = ex.p(z);
    return min_p > 0.0f && p < pmin ? 0ull : ex.mass_of(p);
  };
  u64 mass = 0, kept;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) mass += weight(i);
  block_scan(mass, sm, kept);
  const u64 target = static_cast<u64>(u * static_cast<double>(kept));
  const int token = order_search(sm, a.vocab, target < kept ? target : kept - 1, weight);
  if (threadIdx.x == 0) a.out[r] = token;
}

}  // namespace

const char* sample_rows(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return nullptr;
  if (a.bf16) sample_rows_kernel<__nv_bfloat16><<<a.rows, kThreads, 0, s>>>(a);
  else sample_rows_kernel<float><<<a.rows, kThreads, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace nc
