// Attention of few new tokens per sequence over the paged cache (bf16 or MXFP8 pages): single-token decoding, and chunks
// with up to a few dozen (token, query head) rows per kv head.
//
//   out[row] = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),   s_j = q_row . k_j,  c = scale * log2(e)
//
// Every cached key and value is read once per kv head and used for all rows of its group, so the kernel is bound by
// DRAM. The products run on warp-level tensor-core instructions (m16n8k16) with the 16 keys of a tile on the M side and the rows on
// the N side: eight rows cost what one does, a few percent of the tensor pipe, and neither K nor V goes through shared
// memory in a matrix layout. tcgen05 would need 128-row operands staged by another copy; there is nothing to win at 8.
// The fragment layouts leave the order of the contraction index and of the output channels free, so a lane owns
// contiguous channels: D/4 of a key row for S^T = K Q^T (one MX block for D = 128), D/8 of four value rows for
// O^T = V^T P^T. Each lane copies its own bytes with cp.async into a ring private to its warp and reads back only those:
// no CTA barrier in the main loop. P^T moves from the accumulator to the operand layout by two 8x8 transposes.
//
// grid (key splits, kv heads x row blocks, sequences). Warps of a CTA take 16-key tiles in turn; their partial
// results meet in shared memory, those of different splits in a combine kernel. The reference maximum of a row is raised only
// when a score exceeds it by 2^8 (exact after the division by the sum), so the usual tile needs one vote and no shuffles.
// Probabilities are rounded to bf16 for the second product; the sum is taken of the rounded values, in fp32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "host_build.h"
#include "mx_cache.cuh"
#include "pdl_launch.h"
#include "ptx.cuh"
#include "serving.h"

namespace nc {

namespace {

constexpr int kTile = 16;        // keys per warp step
constexpr int kStages = 3;       // ring depth per warp
constexpr float kRaise = 8.0f;   // log2 units
constexpr float kNoMax = -1.0e30f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? BYTES : 0;   // 0: the destination is filled with zeros
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What the rows [r0, r0 + rows) of sequence b see: row r is query token r / G, head r % G of the kv head's group.
struct Range {
  int n;             // new tokens of the sequence
  int base;          // position of its first new token
  int pmin, pmax;    // positions of the block's first and last real row
  int lo, hi;        // keys [lo, hi) that some row sees; hi <= lo: none
  int tile0, tiles;  // 16-key tiles that cover them
};
__device__ __forceinline__ Range range_of(const PagedAttnArgs& a, int b, int r0, int rows) {
  Range g;
  const int G = a.H / a.KV, len = a.seq_lens[b];
  g.n = a.q_lens != nullptr ? min(max(a.q_lens[b], 0), a.T) : a.T;
  g.base = len - g.n;
  g.lo = g.hi = g.tile0 = g.tiles = 0;
  g.pmin = g.pmax = -1;
  if (r0 >= g.n * G) return g;
  g.pmin = g.base + r0 / G;
  g.pmax = g.base + min((r0 + rows - 1) / G, g.n - 1);
  g.lo = a.window_left >= 0 ? max(0, g.pmin - a.window_left) : 0;
  g.hi = static_cast<int>(min(static_cast<long long>(g.pmax) + 1, static_cast<long long>(a.max_pages) * a.page_size));
  if (g.hi <= g.lo) return g;
  g.tile0 = g.lo / kTile;
  g.tiles = (g.hi + kTile - 1) / kTile - g.tile0;
  return g;
}

template <int D, bool MX>
struct Ring {
  static constexpr int kB = MX ? 1 : 2;                       // bytes per element
  static constexpr int kK = D / 4 * kB, kV = D / 8 * kB;      // bytes a lane owns of one key / value row
  static constexpr int kScale = 16 * (D / 32);                // scale bytes of a tile, one side
  static constexpr int kOffV = 32 * 2 * kK;
  static constexpr int kOffS = kOffV + 32 * 4 * kV;
  static constexpr int kOffPage = kOffS + (MX ? 2 * kScale : 0);
  static constexpr int kStage = (kOffPage + 16 + 15) / 16 * 16;
  static constexpr int kWarps = MX ? 8 : 4;                   // about 100 KB of ring either way: two CTAs per SM
  static constexpr int kBytes = kWarps * kStages * kStage;
};

template <int D, bool MX, int NT>
struct RowsSmem {
  using R = Ring<D, MX>;
  static constexpr int kRows = 8 * NT;
  static constexpr int kTree = R::kWarps / 2 * (D / 16 * NT * 4) * 32 * 4;   // partial sums of half of the warps
  static constexpr int kMain = R::kBytes > kTree ? R::kBytes : kTree;
  static constexpr int kOffML = kMain;
  static constexpr int kTotal = kMain + R::kWarps * kRows * 2 * 4;
};

// P16: page_size is a multiple of 16, so a tile lies in one page.
template <int D, bool MX, int NT, bool P16>
__global__ void __launch_bounds__(Ring<D, MX>::kWarps * 32, NT == 1 ? 2 : 1) paged_rows_kernel(const PagedAttnArgs a) {
  using R = Ring<D, MX>;
  using L = RowsSmem<D, MX, NT>;
  constexpr int W = R::kWarps, ROWS = L::kRows;
  extern __shared__ __align__(16) uint8_t smem[];
  NC_PDL_PROLOGUE();
  const int G = a.H / a.KV;
  const int split = blockIdx.x, kvh = blockIdx.y % a.KV, rb = blockIdx.y / a.KV, b = blockIdx.z;
  const int r0 = rb * ROWS, row_count = min(ROWS, a.T * G - r0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  const Range rg = range_of(a, b, r0, ROWS);
  const int split_tiles = a.split_keys / kTile;
  const int t0 = rg.tile0 + split * split_tiles;
  const int my_tiles = min(rg.tiles - split * split_tiles, split_tiles);
  if (split > 0 && my_tiles <= 0) return;
  if (split == 0 && threadIdx.x == 0 && rg.pmax >= static_cast<long long>(a.max_pages) * a.page_size && a.status != nullptr)
    atomicCAS(a.status, 0, kErrBadIndex);   // keys past the page table are left out
  const float sl = a.scale * 1.4426950408889634f;

  auto q_row = [&](int r) {   // address of row r of the block
    const int t = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
    return a.q + b * a.q_stride_b + t * a.q_stride_t + h * a.q_stride_h;
  };
  // Q as the B operand: row nt * 8 + g8, contraction step s covers channels c * D/4 + 4 s .. + 3
  uint32_t qf[NT][D / 8];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g8;
    const bool ok = r < row_count && (r0 + r) < rg.n * G;
    const __nv_bfloat16* src = ok ? q_row(r) + c * (D / 4) : a.q;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 x = ok ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
      qf[nt][4 * i] = x.x, qf[nt][4 * i + 1] = x.y, qf[nt][4 * i + 2] = x.z, qf[nt][4 * i + 3] = x.w;
    }
  }
  int pos[NT][2];   // positions of the rows this lane holds scores of (accumulator columns 2c, 2c + 1)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + nt * 8 + 2 * c + e;
      pos[nt][e] = r < rg.n * G ? rg.base + r / G : -1;
    }
  // every key of [all_lo, all_hi) is seen by every row of the block
  const int all_lo = a.window_left >= 0 ? max(0, rg.pmax - a.window_left) : 0, all_hi = min(rg.pmin + 1, rg.hi);

  float acc[D / 16][NT][4];
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][nt][e] = 0.0f;
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = kNoMax, l[nt][0] = l[nt][1] = 0.0f;

  uint8_t* ring = smem + warp * (kStages * R::kStage);
  const int count = my_tiles > warp ? (my_tiles - warp + W - 1) / W : 0;
  const int* table = a.page_table + static_cast<long long>(b) * a.max_pages;
  const long long key_stride = static_cast<long long>(a.KV) * D * R::kB;   // bytes
  const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + static_cast<long long>(kvh) * D * R::kB;
  const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + static_cast<long long>(kvh) * D * R::kB;
  const int tiles_per_page = P16 ? a.page_size / kTile : 1;
  int page_ids = -1;   // P16: lane i holds the page of this warp's tile 32 * (block of tiles) + i

  // row (page * page_size + slot) of a key, -1: not in the cache
  auto key_row = [&](int key) -> long long {
    if (key < rg.lo || key >= rg.hi) return -1;
    const int page = table[key / a.page_size];
    return page >= 0 && page < a.num_pages ? static_cast<long long>(page) * a.page_size + key % a.page_size : -1;
  };
  auto issue = [&](int i) {
    uint8_t* st = ring + (i % kStages) * R::kStage;
    const uint32_t dst = smem_u32(st);
    const int tile = t0 + warp + W * i;
    const int key0 = tile * kTile;
    if constexpr (P16) {
      if ((i & 31) == 0) {
        const int mine = t0 + warp + W * (i + lane);
        page_ids = i + lane < count ? table[mine / tiles_per_page] : -1;
      }
      const int page = __shfl_sync(0xffffffffu, page_ids, i & 31);
      const bool page_ok = page >= 0 && page < a.num_pages;
      if (!page_ok && lane == 0 && a.status != nullptr) atomicCAS(a.status, 0, kErrBadIndex);
      const long long row0 = page_ok ? static_cast<long long>(page) * a.page_size + (tile % tiles_per_page) * kTile : 0;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int key = g8 + 8 * hh;
        const bool ok = page_ok && key0 + key >= rg.lo && key0 + key < rg.hi;
        const uint8_t* src = kp + (row0 + key) * key_stride + c * R::kK;
#pragma unroll
        for (int x = 0; x < R::kK / 16; ++x)
          copy_async<16>(dst + ((hh * (R::kK / 16) + x) * 32 + lane) * 16, ok ? src + 16 * x : static_cast<const uint8_t*>(a.k_pool), ok);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 2 * c + (j & 1) + 8 * (j >> 1);
        const bool ok = page_ok && key0 + key >= rg.lo && key0 + key < rg.hi;
        const uint8_t* src = vp + (row0 + key) * key_stride + g8 * R::kV;
        if constexpr (R::kV == 8)
          copy_async<8>(dst + R::kOffV + (j * 32 + lane) * 8, ok ? src : static_cast<const uint8_t*>(a.v_pool), ok);
        else
#pragma unroll
          for (int x = 0; x < R::kV / 16; ++x)
            copy_async<16>(dst + R::kOffV + ((j * (R::kV / 16) + x) * 32 + lane) * 16,
                           ok ? src + 16 * x : static_cast<const uint8_t*>(a.v_pool), ok);
      }
      if constexpr (MX) {   // 16 tokens x D/32 scale bytes of one page and head are contiguous
        constexpr int kLanes = R::kScale / 16;
        if (lane < 2 * kLanes) {
          const bool is_v = lane >= kLanes;
          const int part = is_v ? lane - kLanes : lane;
          const uint8_t* base = is_v ? a.v_scale : a.k_scale;
          const long long off = page_ok ? ((static_cast<long long>(page) * a.KV + kvh) * a.page_size +
                                           (tile % tiles_per_page) * kTile) * (D / 32) + part * 16 : 0;
          copy_async<16>(dst + R::kOffS + (is_v ? R::kScale : 0) + part * 16, base + off, page_ok);
        }
      }
      if (lane == 0) *reinterpret_cast<int*>(st + R::kOffPage) = page_ok;
    } else {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const long long row = key_row(key0 + g8 + 8 * hh);
        const uint8_t* src = kp + row * key_stride + c * R::kK;
#pragma unroll
        for (int x = 0; x < R::kK / 16; ++x)
          copy_async<16>(dst + ((hh * (R::kK / 16) + x) * 32 + lane) * 16,
                         row >= 0 ? src + 16 * x : static_cast<const uint8_t*>(a.k_pool), row >= 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long row = key_row(key0 + 2 * c + (j & 1) + 8 * (j >> 1));
        const uint8_t* src = vp + row * key_stride + g8 * R::kV;
        if constexpr (R::kV == 8)
          copy_async<8>(dst + R::kOffV + (j * 32 + lane) * 8, row >= 0 ? src : static_cast<const uint8_t*>(a.v_pool), row >= 0);
        else
#pragma unroll
          for (int x = 0; x < R::kV / 16; ++x)
            copy_async<16>(dst + R::kOffV + ((j * (R::kV / 16) + x) * 32 + lane) * 16,
                           row >= 0 ? src + 16 * x : static_cast<const uint8_t*>(a.v_pool), row >= 0);
      }
      const int key = key0 + (lane & 15);
      const long long row = key_row(key);
      if (row < 0 && lane < 16 && key >= rg.lo && key < rg.hi && a.status != nullptr) atomicCAS(a.status, 0, kErrBadIndex);
      if constexpr (MX) {
        const uint8_t* base = lane < 16 ? a.k_scale : a.v_scale;
        uint8_t* sd = st + R::kOffS + (lane < 16 ? 0 : R::kScale) + (lane & 15) * (D / 32);
        const long long page = row >= 0 ? row / a.page_size : 0, slot = row >= 0 ? row % a.page_size : 0;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          sd[x] = row >= 0 ? base[((page * a.KV + kvh) * a.page_size + slot) * (D / 32) + x] : 127;
      }
      // validity of the tile's keys, one bit each
      const unsigned bits = __ballot_sync(0xffffffffu, row >= 0);
      if (lane == 0) *reinterpret_cast<int*>(st + R::kOffPage) = static_cast<int>(bits & 0xffffu);
    }
  };

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < count) issue(i);
    copy_commit();
  }
  for (int i = 0; i < count; ++i) {
    copy_wait<kStages - 2>();
    __syncwarp();    // this stage has arrived for every lane; the stage before it has been read by every lane
    if (i + kStages - 1 < count) issue(i + kStages - 1);
    copy_commit();
    const uint8_t* st = ring + (i % kStages) * R::kStage;
    const int key0 = (t0 + warp + W * i) * kTile;
    const int page_info = *reinterpret_cast<const int*>(st + R::kOffPage);
    const bool edge = key0 < all_lo || key0 + kTile > all_hi || (P16 ? page_info == 0 : page_info != 0xffff);
    auto key_ok = [&](int k) {   // key0 + k holds a key of the cache that some row may see
      return key0 + k >= rg.lo && key0 + k < rg.hi && (P16 ? page_info != 0 : ((page_info >> k) & 1) != 0);
    };

    // ---- S^T = K Q^T
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
    uint32_t f1[2], f2[2];
    bool far = false;
    if constexpr (MX) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint32_t sb = st[R::kOffS + (g8 + 8 * hh) * (D / 32) + c * (D / 4) / 32];
        f1[hh] = mx_factor_first(sb) * 0x10001u, f2[hh] = mx_factor_second(sb) * 0x10001u;
        far = far || sb > 134u;
      }
      far = __any_sync(0xffffffffu, far);
    }
#pragma unroll
    for (int x = 0; x < R::kK / 16; ++x) {
      const uint4 w0 = *reinterpret_cast<const uint4*>(st + (x * 32 + lane) * 16);
      const uint4 w1 = *reinterpret_cast<const uint4*>(st + ((R::kK / 16 + x) * 32 + lane) * 16);
      const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
      if constexpr (MX) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t fa[4];
          mx_spread(u0[y], fa[0], fa[2]);
          mx_spread(u1[y], fa[1], fa[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) fa[e] = mul_bf16x2(fa[e], f1[e & 1]);
          if (far) {
#pragma unroll
            for (int e = 0; e < 4; ++e) fa[e] = mul_bf16x2(fa[e], f2[e & 1]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], fa, qf[nt][2 * (4 * x + y)], qf[nt][2 * (4 * x + y) + 1]);
        }
      } else {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t fa[4] = {u0[2 * y], u1[2 * y], u0[2 * y + 1], u1[2 * y + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], fa, qf[nt][2 * (2 * x + y)], qf[nt][2 * (2 * x + y) + 1]);
        }
      }
    }

    // ---- masks, running maximum, probabilities
    if (edge) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = g8 + (e >> 1) * 8, d = pos[nt][e & 1] - (key0 + k);
          if (!(key_ok(k) && d >= 0 && (a.window_left < 0 || d <= a.window_left))) s[nt][e] = -CUDART_INF_F;
        }
    }
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) raise = raise || (s[nt][e] - m[nt][e & 1]) * sl > kRaise;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(m[nt][e], fmaxf(s[nt][e], s[nt][e + 2]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float alpha = fast_exp2((m[nt][e] - mx) * sl);
          m[nt][e] = mx;
          l[nt][e] *= alpha;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) acc[d][nt][e] *= alpha, acc[d][nt][e + 2] *= alpha;
        }
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float c0 = m[nt][0] * sl, c1 = m[nt][1] * sl;
      const uint32_t p0 = pack_bf16(fast_exp2(s[nt][0] * sl - c0), fast_exp2(s[nt][1] * sl - c1));
      const uint32_t p1 = pack_bf16(fast_exp2(s[nt][2] * sl - c0), fast_exp2(s[nt][3] * sl - c1));
      l[nt][0] += bf16_lo(p0) + bf16_lo(p1);
      l[nt][1] += bf16_hi(p0) + bf16_hi(p1);
      pf[nt][0] = transpose_8x8(p0), pf[nt][1] = transpose_8x8(p1);
    }

    // ---- O^T += V^T P^T: keys 2c, 2c + 1 (low, high half of a register) and 2c + 8, 2c + 9
    const uint8_t* sv = st + R::kOffV;
    if constexpr (MX) {
      uint32_t g1[2], g2[2];
      bool vfar = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* ss = st + R::kOffS + R::kScale + (2 * c + 8 * j) * (D / 32) + g8 * (D / 8) / 32;
        uint32_t sa = ss[0], sb = ss[D / 32];
        vfar = vfar || sa > 134u || sb > 134u;
        g1[j] = mx_factor_first(sa) | (mx_factor_first(sb) << 16);
        g2[j] = mx_factor_second(sa) | (mx_factor_second(sb) << 16);
        if (edge) {   // a key outside the cache has codes of zero: its factor must be a number too
          if (!key_ok(2 * c + 8 * j)) g1[j] &= 0xffff0000u, g2[j] &= 0xffff0000u;
          if (!key_ok(2 * c + 8 * j + 1)) g1[j] &= 0xffffu, g2[j] &= 0xffffu;
        }
      }
      vfar = __any_sync(0xffffffffu, vfar);
      constexpr int kWords = R::kV / 4;
      uint32_t v[4][kWords];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kWords == 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(sv + (j * 32 + lane) * 16);
          v[j][0] = w.x, v[j][1] = w.y, v[j][2] = w.z, v[j][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(sv + (j * 32 + lane) * 8);
          v[j][0] = w.x, v[j][1] = w.y;
        }
      }
#pragma unroll
      for (int y = 0; y < kWords; ++y) {
        uint32_t f[2][4];   // [key pair][channel 4y + .], each (first key, second key)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx_spread(__byte_perm(v[2 * j][y], v[2 * j + 1][y], 0x5140), f[j][0], f[j][1]);
          mx_spread(__byte_perm(v[2 * j][y], v[2 * j + 1][y], 0x7362), f[j][2], f[j][3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[j][e] = mul_bf16x2(f[j][e], g1[j]);
          if (vfar) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[j][e] = mul_bf16x2(f[j][e], g2[j]);
          }
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t fa[4] = {f[0][2 * z], f[0][2 * z + 1], f[1][2 * z], f[1][2 * z + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(acc[2 * y + z][nt], fa, pf[nt][0], pf[nt][1]);
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < R::kV / 16; ++x) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(sv + ((j * (R::kV / 16) + x) * 32 + lane) * 16);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t v0 = (&w[0].x)[y], v1 = (&w[1].x)[y], v2 = (&w[2].x)[y], v3 = (&w[3].x)[y];
          const uint32_t fa[4] = {__byte_perm(v0, v1, 0x5410), __byte_perm(v0, v1, 0x7632), __byte_perm(v2, v3, 0x5410),
                                  __byte_perm(v2, v3, 0x7632)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(acc[4 * x + y][nt], fa, pf[nt][0], pf[nt][1]);
        }
      }
    }
  }
  copy_wait<0>();
  __syncthreads();   // the ring is free: it becomes the exchange buffer of the warps

  // ---- the warps' results meet
  float* sm_m = reinterpret_cast<float*>(smem + L::kOffML);
  float* sm_l = sm_m + W * ROWS;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
      if (g8 == 0) {
        sm_m[warp * ROWS + nt * 8 + 2 * c + e] = m[nt][e];
        sm_l[warp * ROWS + nt * 8 + 2 * c + e] = l[nt][e];
      }
    }
  __syncthreads();
  float lt[NT][2], mt[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * c + e;
      float mx = kNoMax;
#pragma unroll
      for (int w = 0; w < W; ++w) mx = fmaxf(mx, sm_m[w * ROWS + r]);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum = fmaf(sm_l[w * ROWS + r], fast_exp2((sm_m[w * ROWS + r] - mx) * sl), sum);
      const float alpha = fast_exp2((m[nt][e] - mx) * sl);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[d][nt][e] *= alpha, acc[d][nt][e + 2] *= alpha;
      lt[nt][e] = sum, mt[nt][e] = mx;
    }
  float* tree = reinterpret_cast<float*>(smem);
  constexpr int kVals = D / 16 * NT * 4;
#pragma unroll
  for (int half = W / 2; half >= 1; half >>= 1) {
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int x = 0; x < kVals; ++x)
        tree[((warp - half) * kVals + x) * 32 + lane] = acc[x / (NT * 4)][(x / 4) % NT][x % 4];
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int x = 0; x < kVals; ++x)
        acc[x / (NT * 4)][(x / 4) % NT][x % 4] += tree[(warp * kVals + x) * 32 + lane];
    }
    __syncthreads();
  }
  if (warp != 0) return;
  const bool whole = rg.tiles <= split_tiles;   // no other split has keys: the result is final
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * c + e;
      if (r >= row_count) continue;
      float f[D / 8];   // channels g8 * D/8 + x
#pragma unroll
      for (int d = 0; d < D / 16; ++d) f[2 * d] = acc[d][nt][e], f[2 * d + 1] = acc[d][nt][e + 2];
      if (whole) {
        const int t = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
        // rows behind the sequence's last new token, and rows that see nothing, are zero
        const float inv = (r0 + r) < rg.n * G && lt[nt][e] > 0.0f ? 1.0f / lt[nt][e] : 0.0f;
        const bool nan = !(lt[nt][e] >= 0.0f);
        __nv_bfloat16* dst = a.out + ((static_cast<long long>(b) * a.T + t) * a.H + h) * D + g8 * (D / 8);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float v0 = f[8 * x + 2 * y], v1 = f[8 * x + 2 * y + 1];
            w[y] = (r0 + r) >= rg.n * G ? 0u : nan ? 0x7fc07fc0u : inv == 0.0f ? 0u : pack_bf16(v0 * inv, v1 * inv);
          }
          *reinterpret_cast<uint4*>(dst + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
        const long long at = (static_cast<long long>(b) * gridDim.y + blockIdx.y) * a.splits + split;
        const int rw = min(ROWS, a.T * G);
        float4* dst = reinterpret_cast<float4*>(a.part_o + (at * rw + r) * D + g8 * (D / 8));
#pragma unroll
        for (int x = 0; x < D / 32; ++x) dst[x] = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
        if (g8 == 0) {
          a.part_ml[(at * rw + r) * 2] = mt[nt][e] * sl;
          a.part_ml[(at * rw + r) * 2 + 1] = lt[nt][e];
        }
      }
    }
}

// One warp per output row: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M). Rows that one split finished are skipped.
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnArgs a, int rows) {
  NC_PDL_PROLOGUE();
  const int G = a.H / a.KV, lane = threadIdx.x & 31;
  const long long total = static_cast<long long>(a.B) * a.KV * a.T * G;
  const long long id = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (id >= total) return;
  const int r = static_cast<int>(id % (a.T * G));
  const int kvh = static_cast<int>(id / (a.T * G) % a.KV), b = static_cast<int>(id / (static_cast<long long>(a.T) * G * a.KV));
  const int rb = r / rows;
  const Range rg = range_of(a, b, rb * rows, rows);
  const int split_tiles = a.split_keys / kTile;
  if (rg.tiles <= split_tiles) return;
  const bool real = r < rg.n * G;   // a row behind the last new token is zero
  const int n = (rg.tiles + split_tiles - 1) / split_tiles;
  const int rw = min(rows, a.T * G);
  const long long blocks = static_cast<long long>(a.KV) * ((a.T * G + rows - 1) / rows);
  const long long at = ((static_cast<long long>(b) * blocks + rb * a.KV + kvh) * a.splits) * rw + (r - rb * rows);
  float mx = -CUDART_INF_F;
  for (int s = lane; real && s < n; s += 32) mx = fmaxf(mx, a.part_ml[(at + static_cast<long long>(s) * rw) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  constexpr int E = D / 32;
  float o[E], ls = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int s = 0; real && s < n; ++s) {
    const long long p = at + static_cast<long long>(s) * rw;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
    const float w = fast_exp2(ml.x - mx);
    ls = fmaf(w, ml.y, ls);
    if constexpr (E == 4) {
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + p * D + lane * 4);
      o[0] = fmaf(w, x.x, o[0]), o[1] = fmaf(w, x.y, o[1]), o[2] = fmaf(w, x.z, o[2]), o[3] = fmaf(w, x.w, o[3]);
    } else {
      const float2 x = *reinterpret_cast<const float2*>(a.part_o + p * D + lane * 2);
      o[0] = fmaf(w, x.x, o[0]), o[1] = fmaf(w, x.y, o[1]);
    }
  }
  const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
  if (!real) {
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
  }
  __nv_bfloat16* dst = a.out + ((static_cast<long long>(b) * a.T + r / G) * a.H + kvh * G + r % G) * D;
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst + lane * 2) = pack_bf16(o[0] * inv, o[1] * inv);
}

// Rows per CTA: the query rows of a kv head in blocks of 8, 16 or 32.
int row_tiles(const PagedAttnArgs& a) {
  const int rows = a.T * (a.H / a.KV);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}

template <int D, bool MX, int NT, bool P16>
cudaError_t launch_rows(const PagedAttnArgs& a, cudaStream_t s) {
  using L = RowsSmem<D, MX, NT>;
  static std::atomic<unsigned long long> configured{0};   // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if ((configured.load(std::memory_order_relaxed) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<D, MX, NT, P16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               L::kTotal);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit);
  }
  const int G = a.H / a.KV, blocks = (a.T * G + L::kRows - 1) / L::kRows;
  cudaError_t e = launch_maybe_pdl(paged_rows_kernel<D, MX, NT, P16>, dim3(a.splits, a.KV * blocks, a.B),
                                   dim3(Ring<D, MX>::kWarps * 32), L::kTotal, s, a);
  if (e != cudaSuccess || a.splits <= 1) return e;
  const long long total = static_cast<long long>(a.B) * a.T * a.H;
  return launch_maybe_pdl(paged_combine_kernel<D>, dim3(static_cast<unsigned>((total + 3) / 4)), dim3(128), 0, s, a,
                          static_cast<int>(L::kRows));
}
template <int D, bool MX>
cudaError_t launch_shape(const PagedAttnArgs& a, cudaStream_t s) {
  const bool p16 = a.page_size % kTile == 0;
#define NC_ROWS(NTV) (p16 ? launch_rows<D, MX, NTV, true>(a, s) : launch_rows<D, MX, NTV, false>(a, s))
  switch (row_tiles(a)) {
    case 1: return NC_ROWS(1);
    case 2: return NC_ROWS(2);
    default: return NC_ROWS(4);
  }
#undef NC_ROWS
}

}  // namespace

PagedPlan paged_rows_plan(const PagedAttnArgs& a) {
  const bool mx = a.k_scale != nullptr;
  const int G = a.H / a.KV, rows = 8 * row_tiles(a), blocks = (a.T * G + rows - 1) / rows;
  const int step = kTile * (mx ? 8 : 4);   // keys that one CTA's warps take at a time
  long long keys = static_cast<long long>(a.max_pages) * a.page_size;
  if (a.window_left >= 0) keys = std::min(keys, static_cast<long long>(a.window_left) + 1 + (rows + G - 1) / G);
  const long long units = static_cast<long long>(a.B) * a.KV * blocks;
  // Two CTAs per SM, twice over, so that sequences of different lengths even out; never less than one step per CTA.
  const long long want = 148 * 4;
  long long per = (keys * units + want - 1) / want;
  per = std::min<long long>((per + step - 1) / step * step, 4096);
  PagedPlan p;
  p.split_keys = static_cast<int>(std::max<long long>(per, step));
  // a range that starts inside a tile touches one tile more
  p.splits = static_cast<int>(((keys + kTile - 1) / kTile + 1 + p.split_keys / kTile - 1) / (p.split_keys / kTile));
  if (p.splits > 1) {
    const long long rw = std::min<long long>(rows, static_cast<long long>(a.T) * G);
    p.part_o = units * p.splits * rw * a.D;
    p.part_ml = units * p.splits * rw * 2;
  }
  return p;
}

const char* paged_rows_attention(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.T == 0) return nullptr;
  if (a.splits > 1 && (a.part_o == nullptr || a.part_ml == nullptr)) return "paged attention: no workspace for the key splits";
  const bool mx = a.k_scale != nullptr;
  const cudaError_t e = a.D == 128 ? (mx ? launch_shape<128, true>(a, s) : launch_shape<128, false>(a, s))
                                   : (mx ? launch_shape<64, true>(a, s) : launch_shape<64, false>(a, s));
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace nc
