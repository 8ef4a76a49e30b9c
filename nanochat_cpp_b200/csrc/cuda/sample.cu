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
// A row belongs to a cluster of 1, 2, 4 or 8 CTAs (more where there are few rows); each copies its slice into shared
// memory, so the logits are read from memory once. A histogram over z (bins of equal width below the maximum: monotone in z, and
// spread, where the bits of z would put most logits into a handful of bins) finds a cut below which nothing can be kept. If at
// most 2048 logits lie above it - the usual settings - they are collected in the first CTA, ranked inside their bins, and
// everything else happens there: only these need the exponential. Otherwise the thresholds are narrowed down by
// further histograms over the bits of z, and the draw walks the vocabulary by halving it among the warps. Bound by the
// chain of such steps (each a pass over the slice and a cluster barrier) for few rows, by 64-bit arithmetic for many.
// Measured (B200): 1 x 65536 top-k 50 top-p 0.95 16 us, 64 x 65536 top-p 0.9 min-p 0.02 26 us, 512 x 32768 bf16 mixed 70 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <atomic>

#include "ptx.cuh"
#include "serving.h"

namespace nc {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kPerThread = kBins / kThreads;
constexpr int kList = 2048;      // candidates that the first CTA ranks in shared memory
constexpr int kMaxCluster = 8;
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

// This CTA's slice of the row: elements [0, n) stand for indices `first` + i. In global memory (RAW) they are as the
// caller left them, in shared memory they have been cleaned.
template <class T, bool RAW>
struct Slice {
  const T* p;
  int n, first;
  __device__ __forceinline__ static float as_is(float z) { return RAW ? clean(z) : z; }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 2) return as_is(__bfloat162float(p[i]));
    else return as_is(p[i]);
  }
  template <class F>
  __device__ __forceinline__ static void spread(const uint4& w, int i, F f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < static_cast<int>(16 / sizeof(T)); ++e) {
      float z;
      if constexpr (sizeof(T) == 2) z = __uint_as_float((e & 1) ? (u[e / 2] & 0xffff0000u) : (u[e / 2] << 16));
      else z = __uint_as_float(u[e]);
      f(i + e, as_is(z));
    }
  }
  // f(i, z) for every element that is not below `floor`, by 16-byte loads between the first and the last aligned address
  template <class F>
  __device__ __forceinline__ void each(float floor, F f) const {
    constexpr int E = 16 / sizeof(T);
    const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int vecs = (n - head) / E;
    auto one = [&](int i, float z) {
      if (z >= floor) f(i, z);
    };
    if (threadIdx.x < head) one(static_cast<int>(threadIdx.x), at(threadIdx.x));
#pragma unroll 2
    for (int v = threadIdx.x; v < vecs; v += kThreads)
      spread(*reinterpret_cast<const uint4*>(p + head + v * E), head + v * E, one);
    for (int i = head + vecs * E + threadIdx.x; i < n; i += kThreads) one(i, at(i));
  }
};

// 2^(j / 32)
__device__ const double kPowers[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// Mass of a logit: exp((z - zmax) / t) in 64 bits, as an integer in units of 2^-fraction. With y = (z - zmax) / t * 32 / ln 2
// split into a whole number k and r in [-1/2, 1/2], p = 2^(k / 32) * 2^(r / 32): the first from a table of 32 and the
// exponent field, the second by its Taylor polynomial to the fourth power (remainder below 2^-39 of p).
struct Exponent {
  double zmax, per;      // per = 32 / (ln 2 * t)
  const double* table;   // shared: 2^(j / 32)
  float z_max, z_cut;    // z_cut: below there is no mass
  int fraction;
  __device__ __forceinline__ double scaled(float z) const {   // p * 2^fraction, z_cut <= z; exactly 2^fraction at the maximum
    constexpr double kShift = 6755399441055744.0;              // 1.5 * 2^52: adding it leaves the whole number in the low bits
    constexpr double kLn = 0.021660849392498290;               // ln 2 / 32
    const double d = static_cast<double>(fminf(z, 3.402823466e38f)) - zmax;
    const double kd = fma(d, per, kShift);
    const int k = __double2loint(kd);
    const double r = fma(d, per, -(kd - kShift));
    const double q = fma(r, fma(r, fma(r, fma(r, kLn * kLn * kLn * kLn / 24, kLn * kLn * kLn / 6), kLn * kLn / 2), kLn), 1.0);
    const double s = table[k & 31];
    return q * __hiloint2double(__double2hiint(s) + (((k >> 5) + fraction) << 20), __double2loint(s));
  }
  __device__ __forceinline__ static u64 whole(double m) {     // round(m), 0 <= m < 2^51
    return static_cast<u64>(__double_as_longlong(m + 4503599627370496.0)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 one() const { return 1ull << fraction; }
  __device__ __forceinline__ u64 mass(float z) const { return z < z_cut ? 0ull : whole(scaled(z)); }
};

struct alignas(16) Shared {
  double table[32];
  union {
    u64 hist[kBins];           // masses or counts of this CTA, summed over the cluster by whoever reads them
    unsigned limb[3][kBins];   // masses in three parts of 16 bits (32-bit additions are native, 64-bit ones a loop)
    struct {                   // the short way, in the first CTA
      u64 sorted[kList], bucket[kThreads];
    };
  };
  u64 list[kList];             // candidates: order key in the high half, ~index in the low
  unsigned count[kBins];       // logits per bin; later, in the first CTA, where the bin's next candidate goes
  u64 warp_sum[kWarps];
  u64 sums[2];                 // this CTA's totals, read by the others (two, used in turn)
  float warp_max[kWarps], warp_min[kWarps];
  int warp_arg[kWarps];
  alignas(16) u64 best[2];                 // of this CTA's slice: largest and smallest logit, index of the largest
  alignas(8) unsigned n;       // candidates collected
  int bin;
  u64 below, inside;
  int lo, hi;
  u64 target;
  int answer;                  // index of a found element, or -1: written by the CTA that has it, into every CTA
  uint32_t cut_key;            // threshold found by the first CTA, written into every CTA
  int cut_last;                // kNoList: too many candidates for the list
};
constexpr int kNoList = -2;
static_assert(sizeof(Shared) <= 49 * 1024, "two CTAs with 64 KB of logits each share an SM");

// What a CTA knows of its cluster, and the steps that need all of it.
struct Cluster {
  int size, rank, turn;
  __device__ __forceinline__ void sync() const {
    if (size > 1) cluster_sync_all();
    else __syncthreads();
  }
  template <class X>
  __device__ __forceinline__ uint32_t peer(const X* x, int r) const { return mapa_u32(x, r); }
};
__device__ __forceinline__ u64 ld_peer_u64(uint32_t at) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_peer_u32(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

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
  const u64 w = warp_scan(lane < kWarps ? sm.warp_sum[lane] : 0, lane);
  total = __shfl_sync(0xffffffffu, w, 31);
  const u64 before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return v + (warp > 0 ? before : 0);
}

// N 64-bit words at `at` in every CTA of the cluster: f(rank, words). Four CTAs' reads are in flight at a time; ranks past
// the cluster read this CTA's own words and are left out by the caller.
template <int N, class F>
__device__ __forceinline__ void read_peers(const Cluster& cl, const u64* at, F f) {
#pragma unroll
  for (int half = 0; half < kMaxCluster; half += 4) {
    if (half >= cl.size) break;
    u64 v[4][N];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t p = cl.peer(at, half + r < cl.size ? half + r : cl.rank);
      if constexpr (N == 1) v[r][0] = ld_peer_u64(p);
      else
#pragma unroll
        for (int i = 0; i < N; i += 2)
          asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v[r][i]), "=l"(v[r][i + 1]) : "r"(p + 8 * i) : "memory");
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) f(half + r, v[r]);
  }
}

// The sum of one value per thread over the cluster; `before` is the part of CTAs of lower rank, `mine` this CTA's.
__device__ __forceinline__ u64 cluster_sum(u64 v, Shared& sm, Cluster& cl, u64& before, u64& mine) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_total(v);
  __syncthreads();
  if (lane == 0) sm.warp_sum[warp] = v;
  __syncthreads();
  mine = warp_total(lane < kWarps ? sm.warp_sum[lane] : 0);
  before = 0;
  if (cl.size == 1) return mine;
  cl.turn ^= 1;   // the slot of the turn before may still be read
  if (threadIdx.x == 0) sm.sums[cl.turn] = mine;
  cl.sync();
  u64 all = 0;
  read_peers<1>(cl, &sm.sums[cl.turn], [&](int r, const u64 (&v)[1]) {
    before += r < cl.rank ? v[0] : 0;
    all += r < cl.size ? v[0] : 0;
  });
  return all;
}

// The bins of all CTAs, kPerThread neighbouring ones per thread.
__device__ __forceinline__ void cluster_bins(Shared& sm, const Cluster& cl, u64 (&x)[kPerThread]) {
  cl.sync();
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) x[i] = cl.size == 1 ? sm.hist[kPerThread * threadIdx.x + i] : 0;
  if (cl.size == 1) return;
  read_peers<kPerThread>(cl, &sm.hist[kPerThread * threadIdx.x], [&](int r, const u64 (&v)[kPerThread]) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) x[i] += r < cl.size ? v[i] : 0;
  });
}
__device__ __forceinline__ void cluster_counts(Shared& sm, const Cluster& cl, const unsigned* bins, u64 (&x)[kPerThread]) {
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) x[i] = cl.size == 1 ? bins[kPerThread * threadIdx.x + i] : 0;
  if (cl.size == 1) return;
  read_peers<kPerThread / 2>(cl, reinterpret_cast<const u64*>(&bins[kPerThread * threadIdx.x]), [&](int r, const u64 (&v)[kPerThread / 2]) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) x[i] += r < cl.size ? (v[i / 2] >> (32 * (i & 1))) & 0xffffffffu : 0;
  });
}

// Candidates that every CTA has collected in its own list, read by the first CTA: f(candidate), each once.
template <class F>
__device__ __forceinline__ void pull_lists(Shared& sm, const Cluster& cl, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = warp % cl.size;   // the warps share out the lists
  const int n = min(static_cast<int>(ld_peer_u64(cl.peer(&sm.n, r)) & 0xffffffffu), kList);
  const uint32_t list = cl.peer(sm.list, r);
#pragma unroll 2
  for (int i = warp / cl.size * 32 + lane; i < n; i += kWarps / cl.size * 32) f(ld_peer_u64(list + 8 * i));
}

// The first index at which the running weight (vocabulary order) exceeds target_of(total weight), or -1; w(i, z) is the
// weight of element i of the slice, 0 below `floor`. The CTA that holds it divides its slice among its warps until one warp can walk it.
template <class S, class Target, class W>
__device__ int order_search(Shared& sm, Cluster& cl, const S& row, float floor, long long* out, Target target_of, W w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = 0, before, mine;
  // the first division is by slices of the CTAs and, inside, by sixteenths for its warps
  int lo = 0, hi = row.n;
  int seg = ((row.n + kWarps - 1) / kWarps + 31) / 32 * 32;
  {
    const int a = min(warp * seg, hi), b = min(a + seg, hi);
    int i = a + lane;
    for (; i + 96 < b; i += 128) {
      float z[4];
      u64 m[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = row.at(i + 32 * e);
      if (!(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])) >= floor)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) m[e] = w(i + 32 * e, z[e]);
      s += (m[0] + m[1]) + (m[2] + m[3]);
    }
    for (; i < b; i += 32) s += w(i, row.at(i));
  }
  u64 target = target_of(cluster_sum(s, sm, cl, before, mine));
  const bool here = target >= before && target - before < mine;
  if (out == nullptr) {
    if (threadIdx.x == 0) sm.answer = -1;
    cl.sync();
  }
  if (here) {
    target -= before;
    for (bool summed = true; hi - lo > 64; summed = false) {
      if (!summed) {
        seg = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
        const int a = min(lo + warp * seg, hi), b = min(a + seg, hi);
        u64 t = 0;
        for (int i = a + lane; i < b; i += 32) t += w(i, row.at(i));
        t = warp_total(t);
        __syncthreads();
        if (lane == 0) sm.warp_sum[warp] = t;
        __syncthreads();
      }
      if (warp == 0) {
        const u64 x = lane < kWarps ? sm.warp_sum[lane] : 0, c = warp_scan(x, lane);
        const unsigned over = __ballot_sync(0xffffffffu, c > target);
        const int f = over ? __ffs(over) - 1 : kWarps - 1;
        if (lane == f) {
          sm.lo = min(lo + f * seg, hi), sm.hi = min(lo + (f + 1) * seg, hi);
          sm.target = target - (c - x);
        }
      }
      __syncthreads();
      lo = sm.lo, hi = sm.hi, target = sm.target;
      __syncthreads();
    }
    if (warp == 0) {
      int found = -1;
      u64 run = 0;
      for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
        const u64 x = i0 + lane < hi ? w(i0 + lane, row.at(i0 + lane)) : 0;
        const u64 c = warp_scan(x, lane) + run;
        const unsigned over = __ballot_sync(0xffffffffu, c > target);
        if (over) found = i0 + __ffs(over) - 1;
        run = __shfl_sync(0xffffffffu, c, 31);
      }
      if (out != nullptr) {
        if (lane == 0) *out = row.first + found;
      } else if (lane < cl.size) {
        const int index = found < 0 ? -1 : row.first + found;
        if (cl.size == 1) sm.answer = index;
        else st_peer_u32(cl.peer(&sm.answer, lane), static_cast<uint32_t>(index));
      }
    }
  }
  if (out != nullptr) {
    if (cl.size > 1) cl.sync();   // no CTA leaves while another reads its shared memory
    return 0;
  }
  cl.sync();
  const int r = sm.answer;
  cl.sync();
  return r;
}

// Kept so far: elements with a key above `key`, and those equal to it up to index `last`.
struct Threshold {
  uint32_t key = 0;
  int last = 0x7fffffff;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

// x: bins of the whole row, from the top. Finds the first bin at which the running weight reaches want_of(total): sm.bin is
// its number (-1: none) and sm.below the weight before it. Returns the running weight before the thread's bins.
template <class Want>
__device__ __forceinline__ u64 first_reaching(Shared& sm, const u64 (&x)[kPerThread], u64 above, Want want_of, u64& total) {
  u64 sum = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) sum += x[i];
  if (threadIdx.x == 0) sm.bin = -1;
  const u64 start = block_scan(sum, sm, total) + above - sum;
  const u64 want = static_cast<u64>(ceil(want_of(total)));   // a whole weight reaches it exactly if it reaches the real number
  u64 c = start;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    if (c < want && c + x[i] >= want) sm.bin = kPerThread * threadIdx.x + i, sm.below = c;
    c += x[i];
  }
  __syncthreads();
  return start;
}

// Descending search among the elements that `in` selects: the largest key at which the running weight (from the top) reaches
// `want` > 0. First over the bins of z, then over the bits of the keys inside the bin. On return sm.below is the
// weight strictly above that key.
template <class S, class Bin, class In, class W>
__device__ uint32_t key_search(Shared& sm, Cluster& cl, const S& row, const Exponent& ex, Bin bin_of, float per, double want, In in, W w) {
  uint32_t lo = order_key(ex.z_cut), hi = order_key(ex.z_max);
  u64 above = 0, total, x[kPerThread];
  int bin = -1;
  for (bool first = true; first || lo < hi; first = false) {
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    cl.sync();   // the bins of the step before have been read by all
    for (int i = threadIdx.x; i < kBins; i += kThreads) sm.hist[i] = 0;
    __syncthreads();
    row.each(ex.z_cut, [&](int i, float z) {
      const uint32_t k = order_key(z);
      if (first) {
        if (in(i, z, k)) atomicAdd(&sm.hist[bin_of(z)], w(z));
      } else if (k >= lo && k <= hi && bin_of(z) == bin && in(i, z, k)) {
        atomicAdd(&sm.hist[(hi - k) >> shift], w(z));
      }
    });
    cluster_bins(sm, cl, x);
    first_reaching(sm, x, above, [&](u64) { return want; }, total);
    const int j = sm.bin;
    const u64 before_j = sm.below;
    __syncthreads();
    if (j >= 0) above = before_j;
    if (j < 0) {      // rounding of `want` past the total: everything is kept
      if (threadIdx.x == 0) sm.below = above + total;
      __syncthreads();
      return lo;
    }
    if (first) {
      // the keys that the bin can hold: a hundredth of a bin more on either side, far above the rounding of bin_of
      bin = j;
      const float z_lo = ex.z_max - (j + 0.51f) / per, z_hi = ex.z_max - (j - 0.51f) / per;
      const bool narrow = per > 0.0f && per < 1e30f;
      if (narrow && z_lo > ex.z_cut && j < kBins - 1) lo = order_key(z_lo);
      if (narrow && z_hi < ex.z_max) hi = order_key(z_hi);
    } else {
      const uint32_t new_hi = hi - (static_cast<uint32_t>(j) << shift);
      const u64 span = (1ull << shift) - 1;
      lo = static_cast<u64>(new_hi) - lo > span ? static_cast<uint32_t>(new_hi - span) : lo;
      hi = new_hi;
    }
  }
  if (threadIdx.x == 0) sm.below = above;
  __syncthreads();
  return lo;
}

template <class T, bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const SampleArgs a, int cluster, int slice) {
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sm = *reinterpret_cast<Shared*>(dyn);
  Cluster cl;
  cl.size = cluster, cl.rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0, cl.turn = 0;
  const int r = blockIdx.x / cluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Slice<T, !STAGED> row;
  row.first = min(cl.rank * slice, a.vocab);
  row.n = min(slice, a.vocab - row.first);
  const Slice<T, true> global{static_cast<const T*>(a.logits) + r * a.ld + row.first, row.n, row.first};
  const float t = a.temperature_rows != nullptr ? a.temperature_rows[r] : a.temperature;
  const float top_p = a.top_p_rows != nullptr ? a.top_p_rows[r] : a.top_p;
  const float min_p = a.min_p_rows != nullptr ? a.min_p_rows[r] : a.min_p;
  int k = a.top_k_rows != nullptr ? a.top_k_rows[r] : a.top_k;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  if (threadIdx.x < 32) sm.table[threadIdx.x] = kPowers[threadIdx.x];
  for (int i = threadIdx.x; i < kBins; i += kThreads) sm.count[i] = 0;
  if (threadIdx.x == 0) sm.n = 0;

  // ---- the largest logit (lowest index of equals) and the smallest above -infinity; the slice goes to shared memory
  // with the alignment that it has, so that 16-byte pieces stay 16-byte pieces
  T* stage = reinterpret_cast<T*>(dyn + (sizeof(Shared) + 15) / 16 * 16) + (reinterpret_cast<uintptr_t>(global.p) & 15) / sizeof(T);
  row.p = STAGED ? stage : global.p;
  float zmax = -CUDART_INF_F, zmin = CUDART_INF_F;
  int arg = 0x7fffffff;
  {
    constexpr int E = 16 / sizeof(T);
    const int head = min(row.n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(global.p) & 15)) & 15) / sizeof(T)));
    const int vecs = (row.n - head) / E;
    auto see = [&](int i, float z) {
      if (z > zmax || (z == zmax && i < arg)) zmax = z, arg = i;
      if (z > -CUDART_INF_F) zmin = fminf(zmin, z);
    };
    auto keep = [&](int i, float z) {
      see(i, z);
      if constexpr (STAGED) stage[i] = static_cast<T>(z);   // (exact: a bf16 value, or fp32)
    };
    if (threadIdx.x < head) keep(threadIdx.x, global.at(threadIdx.x));
#pragma unroll 4
    for (int v = threadIdx.x; v < vecs; v += kThreads) {
      const int i0 = head + v * E;
      uint4 x = __ldcs(reinterpret_cast<const uint4*>(global.p + i0));
      float z[E];
      Slice<T, true>::spread(x, 0, [&](int e, float c) { z[e] = c; });
#pragma unroll
      for (int e = 0; e < E; ++e) see(i0 + e, z[e]);
      if constexpr (STAGED) {
        if constexpr (E == 4)
          x = make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
        else
          x = make_uint4(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]), pack_bf16(z[E - 4], z[E - 3]), pack_bf16(z[E - 2], z[E - 1]));
        *reinterpret_cast<uint4*>(stage + i0) = x;
      }
    }
    for (int i = head + vecs * E + threadIdx.x; i < row.n; i += kThreads) keep(i, global.at(i));
  }
  if (arg != 0x7fffffff) arg += row.first;
  auto take = [&](float oz, int oi, float om) {
    if (oz > zmax || (oz == zmax && oi < arg)) zmax = oz, arg = oi;
    zmin = fminf(zmin, om);
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    take(__shfl_xor_sync(0xffffffffu, zmax, o), __shfl_xor_sync(0xffffffffu, arg, o), __shfl_xor_sync(0xffffffffu, zmin, o));
  if (lane == 0) sm.warp_max[warp] = zmax, sm.warp_arg[warp] = arg, sm.warp_min[warp] = zmin;
  __syncthreads();
  zmax = sm.warp_max[lane % kWarps], arg = sm.warp_arg[lane % kWarps], zmin = sm.warp_min[lane % kWarps];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
    take(__shfl_xor_sync(0xffffffffu, zmax, o), __shfl_xor_sync(0xffffffffu, arg, o), __shfl_xor_sync(0xffffffffu, zmin, o));
  if (cl.size > 1) {
    if (threadIdx.x == 0) {
      sm.best[0] = static_cast<u64>(__float_as_uint(zmax)) << 32 | __float_as_uint(zmin);
      sm.best[1] = static_cast<unsigned>(arg);
    }
    cl.sync();
    read_peers<2>(cl, sm.best, [&](int, const u64 (&v)[2]) {   // (this CTA's own again where the cluster is smaller)
      take(__uint_as_float(static_cast<uint32_t>(v[0] >> 32)), static_cast<int>(v[1]), __uint_as_float(static_cast<uint32_t>(v[0])));
    });
  }
  if (zmax == -CUDART_INF_F || !(t > 0.0f) || k == 1 || !(top_p > 0.0f) || !(min_p <= 1.0f)) {
    if (threadIdx.x == 0 && cl.rank == 0) a.out[r] = zmax == -CUDART_INF_F ? -1 : arg;
    if (cl.size > 1) cl.sync();   // no CTA leaves while another reads its shared memory
    return;
  }
  Exponent ex;
  ex.zmax = static_cast<double>(fminf(zmax, 3.402823466e38f)), ex.z_max = zmax, ex.table = sm.table;
  ex.per = 46.166241308446828384 / static_cast<double>(t);
  int log_v = 0;
  while ((1ll << log_v) < a.vocab) ++log_v;
  ex.fraction = min(46, 62 - log_v);
  // -infinity has no mass at any temperature, and neither has anything beside +infinity
  ex.z_cut = zmax == CUDART_INF_F ? zmax : fmaxf(zmax - kReach * t, -3.402823466e38f);
  const double u = fmax(static_cast<double>(a.u[r]), 0.0), want_p = static_cast<double>(top_p);
  const double pmin = static_cast<double>(min_p) * static_cast<double>(ex.one());   // in units of mass
  const bool nucleus = top_p < 1.0f, filtered = k < a.vocab || nucleus || min_p > 0.0f;

  Threshold cut;                    // what top-k and top-p keep, when the long way is taken
  cut.key = order_key(ex.z_cut);
  float floor = ex.z_cut;           // nothing below has a mass that counts
  if (filtered) {
    const float width = fminf(zmax - zmin, kReach * t);
    const float per = width > 0.0f ? fminf(static_cast<float>(kBins) / width, 1e37f) : 0.0f;
    // the nearest whole number to (zmax - z) * per, left in the low bits by adding 2^23. A difference that overflows goes to the last
    // bin (as NaN where `per` is 0: fminf takes the other operand).
    auto bin_of = [&](float z) { return __float_as_int(fminf(fmaf(zmax - z, per, 8388608.0f), 8388608.0f + (kBins - 1))) & 0x7fffff; };
    row.each(ex.z_cut, [&](int, float z) { atomicAdd(&sm.count[bin_of(z)], 1u); });
    cl.sync();
    u64 x[kPerThread], total;
    cluster_counts(sm, cl, sm.count, x);
    // the first bin at which k logits are reached, and the last one that min_p can keep anything of
    const u64 start = first_reaching(sm, x, 0, [&](u64) { return static_cast<double>(k); }, total);
    const int bin_k = sm.bin < 0 ? kBins - 1 : sm.bin;
    const u64 above_k = sm.bin < 0 ? 0 : sm.below;
    int bin_m = kBins - 1;
    if (min_p > 0.0f) {   // rounded down generously; the exact comparison follows
      const float z = zmax + t * logf(min_p) * 1.0001f - 1e-5f * (fabsf(zmax) + 1.0f);
      bin_m = z > ex.z_cut ? bin_of(z) : kBins - 1;
    }
    const int bin_cut = min(bin_k, bin_m);
    u64 c = start;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      c += x[i];
      if (static_cast<int>(kPerThread * threadIdx.x) + i == bin_cut) sm.inside = c;
    }
    cl.sync();
    const u64 n_cut = sm.inside;

    if (n_cut <= kList) {
      // ---- the short way, in the first CTA: candidates go to their bin's places, are ranked inside it, and decided on
      const float z_lo = bin_cut < kBins - 1 && per > 0.0f && per < 1e30f ? fmaxf(zmax - (bin_cut + 0.51f) / per, ex.z_cut) : ex.z_cut;
      row.each(z_lo, [&](int i, float z) {
        if (bin_of(z) > bin_cut) return;
        sm.list[atomicAdd(&sm.n, 1u)] = (static_cast<u64>(order_key(z)) << 32) | static_cast<uint32_t>(~(row.first + i));
      });
      if (cl.rank == 0) {
        c = start;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) sm.count[kPerThread * threadIdx.x + i] = static_cast<unsigned>(c), c += x[i];
      }
      cl.sync();
      if (cl.rank == 0)
        pull_lists(sm, cl, [&](u64 e) {
          sm.sorted[atomicAdd(&sm.count[bin_of(key_value(static_cast<uint32_t>(e >> 32)))], 1u)] = e;
        });
      cl.sync();
      if (cl.rank != 0) return;   // nobody reads this CTA's memory any more
      const int n = static_cast<int>(n_cut);
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 e = sm.sorted[i];
        const int bin = bin_of(key_value(static_cast<uint32_t>(e >> 32)));
        const int from = bin > 0 ? sm.count[bin - 1] : 0, to = sm.count[bin];   // where the bin before, and this one, ends
        int rank = from;
        for (int j = from; j < to; ++j) rank += sm.sorted[j] > e;
        sm.list[rank] = e;
      }
      sm.bucket[threadIdx.x] = 0;
      if (threadIdx.x == 0) sm.n = 0;
      __syncthreads();
      // two neighbours per thread
      constexpr int N = kList / kThreads;
      u64 mine[N], sum = 0, total_k;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = N * threadIdx.x + e;
        mine[e] = 0;
        if (i < n && i < k) {
          const float z = key_value(static_cast<uint32_t>(sm.list[i] >> 32));
          const double p = ex.scaled(z);
          if (i == 0 || p >= pmin) mine[e] = Exponent::whole(p);
        }
        sum += mine[e];
      }
      u64 before = block_scan(sum, sm, total_k) - sum;
      // Back to vocabulary order: the mass of each of kThreads ranges of indices, the range in which the draw falls,
      // and the few candidates inside it.
      const unsigned range = (a.vocab + kThreads - 1) / kThreads;
      uint32_t index[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = N * threadIdx.x + e;
        if (nucleus && i > 0 && static_cast<double>(before) >= want_p * static_cast<double>(total_k)) mine[e] = 0;
        else before += mine[e];
        index[e] = i < n ? ~static_cast<uint32_t>(sm.list[i]) : 0;
        if (mine[e] > 0) atomicAdd(&sm.bucket[index[e] / range], mine[e]);
      }
      __syncthreads();
      const u64 here = sm.bucket[threadIdx.x];
      u64 kept;
      const u64 upto = block_scan(here, sm, kept);
      const u64 target = static_cast<u64>(u * static_cast<double>(kept)), goal = target < kept ? target : kept - 1;
      if (upto > goal && upto - here <= goal) sm.bin = threadIdx.x, sm.below = upto - here;
      __syncthreads();
      const unsigned bucket = sm.bin;
      const u64 base = sm.below;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (mine[e] > 0 && index[e] / range == bucket) {
          sm.sorted[atomicAdd(&sm.n, 1u)] = (static_cast<u64>(index[e]) << 32) | static_cast<unsigned>(N * threadIdx.x + e);
        }
      __syncthreads();
      const int members = static_cast<int>(sm.n);   // index in the high half, place in the list in the low
      auto mass_of = [&](u64 m) { return ex.mass(key_value(static_cast<uint32_t>(sm.list[static_cast<uint32_t>(m)] >> 32))); };
      for (int i = threadIdx.x; i < members; i += kThreads) {
        u64 cum = base;
        for (int j = 0; j < members; ++j)
          if (sm.sorted[j] < sm.sorted[i]) cum += mass_of(sm.sorted[j]);
        if (cum <= goal && cum + mass_of(sm.sorted[i]) > goal) a.out[r] = static_cast<long long>(sm.sorted[i] >> 32);
      }
      return;
    }

    // ---- the long way: thresholds by histograms of counts and masses
    if (bin_m < kBins - 1 && per > 0.0f && per < 1e37f) floor = fmaxf(floor, zmax - (bin_m + 0.51f) / per);   // min_p keeps nothing below
    if (above_k < static_cast<u64>(k) && total > static_cast<u64>(k)) {
      const uint32_t key = key_search(sm, cl, row, ex, bin_of, per, static_cast<double>(k), [](int, float, uint32_t) { return true; },
                                      [](float) { return 1ull; });
      const u64 ties = static_cast<u64>(k) - sm.below;   // that many of the equals are kept
      __syncthreads();
      cut.key = key;
      floor = fmaxf(floor, key_value(key));
      cut.last = order_search(sm, cl, row, key_value(key), nullptr, [&](u64) { return ties - 1; }, [&](int, float z) { return order_key(z) == key ? 1ull : 0ull; });
      if (cut.last < 0) cut.last = 0x7fffffff;
    }
    if (nucleus) {
      const Threshold top = cut;
      auto mass_in = [&](int i, float z) {   // of an element that top-k and min_p keep; no branches, so that several overlap
        const bool keep = z >= ex.z_cut && top.keeps(order_key(z), row.first + i);
        const double p = ex.scaled(fmaxf(z, ex.z_cut));
        const u64 m = Exponent::whole(p);
        return keep && p >= pmin ? m : 0ull;
      };
      double want = 0.0;
      u64 all = 0;
      int j = -1;
      if (slice <= 65536) {   // a part of 16 bits cannot overflow 32
        cl.sync();
        for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sm.limb[0][0])[i] = 0;
        __syncthreads();
        row.each(floor, [&](int i, float z) {
          const u64 m = mass_in(i, z);
          if (m == 0) return;
          const int bin = bin_of(z);
          atomicAdd(&sm.limb[0][bin], static_cast<unsigned>(m) & 0xffffu);
          atomicAdd(&sm.limb[1][bin], static_cast<unsigned>(m >> 16) & 0xffffu);
          atomicAdd(&sm.limb[2][bin], static_cast<unsigned>(m >> 32));
        });
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {   // the parts make whole masses again, in the same memory
          const int bin = kPerThread * threadIdx.x + i;
          x[i] = (static_cast<u64>(sm.limb[2][bin]) << 32) + (static_cast<u64>(sm.limb[1][bin]) << 16) + sm.limb[0][bin];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) sm.hist[kPerThread * threadIdx.x + i] = x[i];
        cluster_bins(sm, cl, x);
        first_reaching(sm, x, 0, [&](u64 sum) { return want = want_p * static_cast<double>(sum); }, all);
        j = sm.bin;
        const u64 above = sm.below;
        __syncthreads();
        // the bin's elements, ranked in the first CTA: the last one with less than `want` before it is the last to be kept
        if (j >= 0) {
          const bool narrow = per > 0.0f && per < 1e30f;   // (bounds a hundredth of a bin wide of it)
          const float z_lo = narrow && j < kBins - 1 ? fmaxf(zmax - (j + 0.51f) / per, ex.z_cut) : ex.z_cut;
          const float z_hi = narrow && j > 0 ? zmax - (j - 0.51f) / per : zmax;
          row.each(z_lo, [&](int i, float z) {
            if (z > z_hi || bin_of(z) != j || mass_in(i, z) == 0) return;
            const unsigned at = atomicAdd(&sm.n, 1u);
            if (at < static_cast<unsigned>(kList))
              sm.list[at] = (static_cast<u64>(order_key(z)) << 32) | static_cast<uint32_t>(~(row.first + i));
          });
          cl.sync();
          if (cl.rank == 0) {
            u64 n_all = 0;
            read_peers<1>(cl, reinterpret_cast<const u64*>(&sm.n),
                          [&](int c, const u64 (&v)[1]) { n_all += c < cl.size ? v[0] & 0xffffffffu : 0; });
            const int n = static_cast<int>(n_all);
            if (threadIdx.x == 0) sm.cut_last = kNoList, sm.lo = 0;
            __syncthreads();
            if (n_all <= kList) {
              pull_lists(sm, cl, [&](u64 e) { sm.sorted[atomicAdd(&sm.lo, 1)] = e; });
              __syncthreads();
              for (int i = threadIdx.x; i < n; i += kThreads) {
                const u64 e = sm.sorted[i];
                int rank = 0;
                for (int o = 0; o < n; ++o) rank += sm.sorted[o] > e;
                sm.list[rank] = e;
              }
              __syncthreads();
              constexpr int N = kList / kThreads;
              u64 mine[N], sum = 0, dummy;
#pragma unroll
              for (int e = 0; e < N; ++e) {
                const int i = N * threadIdx.x + e;
                mine[e] = i < n ? ex.mass(key_value(static_cast<uint32_t>(sm.list[i] >> 32))) : 0;
                sum += mine[e];
              }
              u64 before = block_scan(sum, sm, dummy) - sum + above;
#pragma unroll
              for (int e = 0; e < N; ++e) {
                const int i = N * threadIdx.x + e;
                const bool keep = i < n && static_cast<double>(before) < want;
                before += mine[e];
                const bool next = i + 1 < n && static_cast<double>(before) < want;
                if (keep && !next) {
                  sm.cut_key = static_cast<uint32_t>(sm.list[i] >> 32);
                  sm.cut_last = static_cast<int>(~static_cast<uint32_t>(sm.list[i]));
                }
              }
            }
            __syncthreads();
            if (threadIdx.x > 0 && static_cast<int>(threadIdx.x) < cl.size) {
              st_peer_u32(cl.peer(&sm.cut_key, threadIdx.x), sm.cut_key);
              st_peer_u32(cl.peer(&sm.cut_last, threadIdx.x), static_cast<uint32_t>(sm.cut_last));
            }
          }
          cl.sync();
          if (sm.cut_last != kNoList) cut.key = sm.cut_key, cut.last = sm.cut_last;
          else j = -2;   // more equal or nearly equal logits than the list holds
        }
      } else {
        j = -2;
      }
      if (j == -2) {
        auto in = [&](int i, float z, uint32_t) { return mass_in(i, z) > 0; };
        u64 mass = 0, b, m;
        row.each(floor, [&](int i, float z) { mass += mass_in(i, z); });
        all = cluster_sum(mass, sm, cl, b, m);
        want = want_p * static_cast<double>(all);
        const uint32_t key = key_search(sm, cl, row, ex, bin_of, per, want, in, [&](float z) { return ex.mass(z); });
        const u64 above = sm.below, each = ex.mass(key_value(key));
        __syncthreads();
        if (above < all) {   // (else rounding took `want` past the total: nothing is cut)
          // equals are kept while the mass before them is short of `want`
          const double need = each > 0 ? ceil((want - static_cast<double>(above)) / static_cast<double>(each)) : 1.0;
          u64 ties = need < 1.0 ? 1 : static_cast<u64>(need);
          while (ties > 1 && static_cast<double>(above + (ties - 1) * each) >= want) --ties;
          while (static_cast<double>(above + ties * each) < want && ties < static_cast<u64>(a.vocab)) ++ties;
          const int last = order_search(sm, cl, row, key_value(key), nullptr, [&](u64) { return ties - 1; }, [&](int i, float z) {
            return order_key(z) == key && top.keeps(key, row.first + i) ? 1ull : 0ull;
          });
          if (last >= 0) cut.last = last;
          else if (key != top.key) cut.last = 0x7fffffff;
          cut.key = key;
        }
      }
    }
  }

  // ---- the draw, over the vocabulary
  floor = fmaxf(floor, key_value(cut.key));
  order_search(sm, cl, row, floor, a.out + r,
               [&](u64 kept) {
                 const u64 target = static_cast<u64>(u * static_cast<double>(kept));
                 return target < kept ? target : kept - 1;
               },
               [&](int i, float z) {
                 const bool keep = z >= ex.z_cut && cut.keeps(order_key(z), row.first + i);
                 const double p = ex.scaled(fmaxf(z, ex.z_cut));
                 const u64 m = Exponent::whole(p);
                 return keep && p >= pmin ? m : 0ull;
               });
}

template <class T>
cudaError_t launch_sample(const SampleArgs& a, cudaStream_t s) {
  // Enough CTAs for two per SM where rows are few, and slices that leave room for two CTAs' on an SM; a vocabulary that
  // does not fit eight SMs' shared memory is read from global memory in every pass.
  constexpr int kFixed = (sizeof(Shared) + 15) / 16 * 16 + 16, kHalf = 113 * 1024, kWhole = 227 * 1024;
  int c = 1;
  while (c < kMaxCluster && (static_cast<long long>(a.rows) * c < 148 || static_cast<long long>(a.vocab) * sizeof(T) / c > kHalf - kFixed - 64)) c *= 2;
  constexpr int E = 16 / sizeof(T);
  const int slice = static_cast<int>(((static_cast<long long>(a.vocab) + c - 1) / c + E - 1) / E * E);
  const bool staged = static_cast<long long>(slice) * sizeof(T) + kFixed <= kWhole;
  const size_t smem = kFixed + (staged ? static_cast<size_t>(slice) * sizeof(T) : 0);
  static std::atomic<unsigned long long> configured{0};   // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if ((configured.load(std::memory_order_relaxed) & bit) == 0) {
    cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWhole);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(sample_rows_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWhole);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, staged ? sample_rows_kernel<T, true> : sample_rows_kernel<T, false>, a, c, slice);
}

}  // namespace

const char* sample_rows(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return nullptr;
  if (static_cast<long long>(a.rows) * kMaxCluster >= (1LL << 31)) return "sample_rows: too many rows";
  const cudaError_t e = a.bf16 ? launch_sample<__nv_bfloat16>(a, s) : launch_sample<float>(a, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace nc
