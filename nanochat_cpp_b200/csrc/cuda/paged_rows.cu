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
// O^T = V^T P^T. Rows arrive by cp.async, whole rows per instruction (lanes that took their own quarter row asked L2
// for every 32-byte sector twice), in a ring private to the warp: no CTA barrier in the main loop. P^T moves from the accumulator to the operand layout by two 8x8 transposes.
//
// A warp is a unit of its own: it takes one run of keys (`split_keys`) of one sequence, kv head and block of rows, and
// writes its partial sums; a combine kernel joins the runs of a row. Nothing in the CTA waits for anything else, and
// sequences of different lengths even out over many equal units. The reference maximum of a row is raised only when a
// score exceeds it by 2^8 or 2^7 (exact after the division by the sum), so the usual tile needs one vote and no shuffles.
// Probabilities are rounded to 16 bits for the second product; the sum is taken of the rounded values, in fp32. On MXFP8 pages
// the products run in f16, which takes E4M3 codes in one instruction a pair and probabilities to 11 bits (and to 2^-32 of the
// reference). A run whose blocks, or whose queries' channels, lie further apart than f16 reaches is walked again in bf16: where all
// are, 64 sequences of 2000 keys take 121 us instead of 88, 32 of 20000 236 instead of 172.
// Measured (B200, MXFP8, D = 128): 64 sequences up to 2048 keys 50..51 us (3.4 TB/s), 32 up to 32768 173..181 us (4.9..5.1 TB/s);
// 64 x 4 new tokens over bf16 71 us (4.9 TB/s).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "host_build.h"
#include "mx_cache.cuh"
#include "paged_common.cuh"
#include "pdl_launch.h"
#include "ptx.cuh"
#include "serving.h"

namespace nc {

namespace {

constexpr int kTile = 16;        // keys per warp step
constexpr int kStages = 3;       // ring depth per warp
constexpr int kPart = 512;       // keys of a run whose page numbers are at hand, one per lane: a longer run goes part by part
constexpr float kNoMax = -1.0e30f;
constexpr int kReach = 14;       // powers of two from the largest scale to one that is a normal f16: its codes are exact there
constexpr int kUnset = -1000;    // no reference yet: out of reach of every scale byte
constexpr int kClimb = 45;       // that the scale of the values' sums may grow by before what was summed first would lose bits

template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two E4M3 codes (the low or the high half of w) as f16: exact
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// 2^(b - 127) of a scale byte, or of kUnset (any finite number)
__device__ __forceinline__ float scale_value(int b) { return __uint_as_float(b > 0 ? static_cast<uint32_t>(b) << 23 : 0x00400000u); }
// 2^d for d <= 0 (0 below the range of fp32)
__device__ __forceinline__ float pow2_neg(int d) { return __uint_as_float(static_cast<uint32_t>(max(127 + d, 0)) << 23); }
// of each half the smaller magnitude (its sign means nothing)
__device__ __forceinline__ uint32_t min_magnitude_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
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

template <int D, bool MX>
struct Ring {
  static constexpr int kRow = D * (MX ? 1 : 2);               // bytes of a key or value row
  static constexpr int kLanes = kRow / 16;                    // lanes that copy one row
  static constexpr int kCopies = 16 * kLanes / 32;            // copies per lane and side
  static constexpr int kScale = 16 * (D / 32);                // scale bytes of a tile, one side
  static constexpr int kOffV = 16 * kRow;
  static constexpr int kOffS = 2 * kOffV;
  static constexpr int kOffPage = kOffS + (MX ? 2 * kScale : 0);   // which keys are usable, where a tile spans pages
  static constexpr int kStage = kOffPage + 16;
  static constexpr int kBytes = kStages * kStage;
  // Place of 16-byte piece `p` of row `key` inside the row, chosen so that the eight lanes of a 16-byte read phase hit
  // different banks: they read pieces of keys (0, 1) at distance kRow / 64 on the key side, and pieces (0, 1) times
  // kRow / 128 of keys 0, 2, 4, 6 on the value side.
  static __device__ __forceinline__ int place_k(int key, int p) {
    if constexpr (kRow == 256) return p ^ ((p >> 3) + 2 * (key & 1));
    else if constexpr (kRow == 128) return p ^ (key & 1);
    else return p;
  }
  static __device__ __forceinline__ int place_v(int key, int p) {
    if constexpr (kRow == 256) return p ^ (4 * ((key >> 1) & 1) + ((key >> 2) & 1));
    else if constexpr (kRow == 128) return p ^ (2 * ((key >> 1) & 3));
    else return p ^ ((key >> 1) & 3);
  }
};

// One run of keys. P16: page_size is a multiple of 16, so a tile lies in one page. F16 (MXFP8 pages): the products run in f16, on codes
// and powers of two, which is exact while the numbers fit it; where they do not, nothing has been written and the answer is
// false. Without F16 they run in bf16, which holds every value of either cache.
template <int D, bool MX, bool F16, int NT, bool P16>
__device__ __forceinline__ bool walk(const PagedAttnArgs& a, uint8_t* smem) {
  using R = Ring<D, MX>;
  constexpr int ROWS = 8 * NT;
  // By how much a score may exceed its row's reference, in log2 units. In f16 (below 2^16) probabilities are taken 2^7 times too large,
  // and where scores are so large that fp32 steps by 8, "7 below the reference" is 8 below it: 2^15 at most.
  constexpr float kRaise = F16 ? 7.0f : 8.0f;
  const int G = a.H / a.KV;
  const int lane = threadIdx.x, g8 = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y % a.KV, rb = blockIdx.y / a.KV, b = blockIdx.z;
  const int r0 = rb * ROWS, row_count = min(ROWS, a.T * G - r0);
  const Range rg = range_of(a, b, r0, ROWS, kTile);
  const int split_tiles = a.split_keys / kTile;
  int t0 = rg.tile0 + split * split_tiles, left = min(rg.tiles - split * split_tiles, split_tiles);
  if (split > 0 && left <= 0) return true;
  int count = min(left, kPart / kTile);   // tiles of the part that begins at tile t0
  if (split == 0 && lane == 0 && rg.pmax >= static_cast<long long>(a.max_pages) * a.page_size && a.status != nullptr)
    atomicCAS(a.status, 0, kErrBadIndex);   // keys past the page table are left out
  const float sl = a.scale * 1.4426950408889634f;

  auto q_row = [&](int r) {   // address of row r of the block
    const int t = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
    return a.q + b * a.q_stride_b + t * a.q_stride_t + h * a.q_stride_h;
  };
  // Q as the B operand: row nt * 8 + g8, contraction step s covers channels c * D/4 + 4 s .. + 3. For f16 a row of Q is brought
  // below 2^15 by a power of two, which goes into the row's score factor: exact if its smallest nonzero magnitude lies no more
  // than 31 powers of two below the largest (bf16's 8 bits then end at f16's last step, 2^-24, or before). Rows with a
  // result below 2^-17, zeros among them, are looked at again when the first keys have been asked for.
  uint32_t qf[NT][D / 8];
  float row_factor[NT];
  bool tiny = false;
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
    row_factor[nt] = sl;
    if constexpr (F16) {
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) mx = __vmaxu2(mx, qf[nt][i] & 0x7fff7fffu);
      mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const uint32_t top = max(mx & 0xffffu, mx >> 16);
      int e = static_cast<int>(top >> 7);                  // biased exponent of the largest magnitude
      if (top == 0 || top >= 0x7f80) e = 127 + 14;         // nothing to scale: zeros, infinities, NaN
      e = max(e, 15);
      const float up = __uint_as_float(static_cast<uint32_t>(min(127 + 14 + 127 - e, 254)) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(max(e - 14, 1)) << 23);
      uint32_t least = 0x7c007c00u;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        qf[nt][i] = pack_f16(bf16_lo(qf[nt][i]) * up, bf16_hi(qf[nt][i]) * up);
        least = min_magnitude_f16x2(least, qf[nt][i]);
      }
      row_factor[nt] = down * sl;
      tiny = tiny || (ok && min(least & 0x7fffu, (least >> 16) & 0x7fffu) < 0x80u);
    }
  }
  float factor[NT][2];   // score factor of the rows this lane holds scores of (accumulator columns 2c, 2c + 1)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) factor[nt][e] = __shfl_sync(0xffffffffu, row_factor[nt], (2 * c + e) * 4);
  int pos[NT][2];        // and their positions
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
  float m[NT][2];        // reference maximum, in units of the exponent
  float l[NT][4];        // sums of the rounded probabilities: P^T times a row of ones on the tensor core
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = kNoMax, l[nt][0] = l[nt][1] = l[nt][2] = l[nt][3] = 0.0f;
  // Codes enter the f16 products as code * 2^(b - ref): exact while b lies no more than kReach below ref, the largest scale
  // byte of the tile's usable keys or more (keys), of the run's usable values so far (values). The scores take 2^(k_ref - 127)
  // into their factor; a larger v_ref scales down what has been summed.
  int k_ref = kUnset, v_ref = kUnset, v_first = kUnset;
  float k_unit = 1.0f;

  uint8_t* ring = smem;
  const int* table = a.page_table + static_cast<long long>(b) * a.max_pages;
  const uint32_t stride = static_cast<uint32_t>(a.KV) * R::kRow;   // bytes from a token to the next
  // what this lane copies: piece lane % kLanes of rows lane / kLanes, and every 32 / kLanes-th after it
  const int row_l = lane / R::kLanes, piece = lane % R::kLanes;
  constexpr int kStep = 32 / R::kLanes;
  const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + kvh * R::kRow + piece * 16;
  const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + kvh * R::kRow + piece * 16;
  // and reads: its quarter of key row g8, its eighth of value row 2c
  int k_at[R::kRow / 64], v_at[R::kRow >= 128 ? R::kRow / 128 : 1];
#pragma unroll
  for (int x = 0; x < R::kRow / 64; ++x) k_at[x] = g8 * R::kRow + R::place_k(g8, c * (R::kRow / 64) + x) * 16;
  if constexpr (R::kRow >= 128) {
#pragma unroll
    for (int x = 0; x < R::kRow / 128; ++x) v_at[x] = R::kOffV + 2 * c * R::kRow + R::place_v(2 * c, g8 * (R::kRow / 128) + x) * 16;
  } else {
    v_at[0] = R::kOffV + 2 * c * R::kRow + R::place_v(2 * c, g8 / 2) * 16 + (g8 & 1) * 8;
  }
  // P16: lane i holds the i-th page of the part, and `at_page`, `in_page` follow the tiles that are requested
  const int tiles_per_page = P16 ? a.page_size / kTile : 1;
  int page_ids = -1, at_page = 0, in_page = 0;
  unsigned bad_tiles = 0;   // P16: bit i: the page of tile i is unmapped or outside the pool
  auto look_up = [&]() {
    const int first = t0 / tiles_per_page;
    at_page = 0, in_page = t0 - first * tiles_per_page, page_ids = -1;
    if (count > 0 && first + lane <= (t0 + count - 1) / tiles_per_page) page_ids = table[first + lane];
    const int mine = __shfl_sync(0xffffffffu, page_ids, (in_page + lane) / tiles_per_page);
    bad_tiles = __ballot_sync(0xffffffffu, lane < count && (mine < 0 || mine >= a.num_pages));
    if (bad_tiles != 0 && lane == 0 && a.status != nullptr) atomicCAS(a.status, 0, kErrBadIndex);
  };
  if constexpr (P16) look_up();
  const uint8_t* s_lane = nullptr;
  uint32_t s_dst = 0, s_stride = 0;
  constexpr int kScaleLanes = MX ? R::kScale / 16 : 1;   // 16-byte pieces of a tile's scales, one side
  if constexpr (MX) {
    const int part = lane % kScaleLanes;
    const bool is_v = lane >= kScaleLanes;
    s_lane = (is_v ? a.v_scale : a.k_scale) + static_cast<long long>(kvh) * a.page_size * (D / 32) + part * 16;
    s_dst = R::kOffS + (is_v ? R::kScale : 0) + part * 16;
    s_stride = static_cast<uint32_t>(a.KV * a.page_size * (D / 32));
  }

  // row (page * page_size + slot) of a key, -1: not in the cache
  auto key_row = [&](int key) -> long long {
    if (key < rg.lo || key >= rg.hi) return -1;
    const int page = table[key / a.page_size];
    return page >= 0 && page < a.num_pages ? static_cast<long long>(page) * a.page_size + key % a.page_size : -1;
  };
  int put = 0, get = 0;   // stages that are written and read next
  auto issue = [&](int i) {
    uint8_t* st = ring + put * R::kStage;
    put = put + 1 == kStages ? 0 : put + 1;
    const uint32_t dst = smem_u32(st);
    const int key0 = (t0 + i) * kTile;
    if constexpr (P16) {
      // a page that is none of the pool's stands for page 0: its rows are requested as zeros
      const bool page_ok = ((bad_tiles >> i) & 1) == 0;
      const int id = __shfl_sync(0xffffffffu, page_ids, at_page);
      const uint32_t page = page_ok ? id : 0, slot0 = in_page * kTile;
      if (++in_page == tiles_per_page) in_page = 0, ++at_page;
      // all 16 rows lie inside the page, wanted or not
      const unsigned long long base = (static_cast<unsigned long long>(page) * a.page_size + slot0 + row_l) * stride;
      const uint8_t *ks = kp + base, *vs = vp + base;
      auto rows_in = [&](auto wanted) {
#pragma unroll
        for (int x = 0; x < R::kCopies; ++x) {
          const int key = row_l + x * kStep;
          const bool ok = wanted(key);
          copy_async<16>(dst + key * R::kRow + R::place_k(key, piece) * 16, ks + x * kStep * stride, ok);
          copy_async<16>(dst + R::kOffV + key * R::kRow + R::place_v(key, piece) * 16, vs + x * kStep * stride, ok);
        }
      };
      if (page_ok && key0 >= rg.lo && key0 + kTile <= rg.hi) rows_in([](int) { return true; });
      else rows_in([&](int k) { return page_ok && key0 + k >= rg.lo && key0 + k < rg.hi; });
      if constexpr (MX) {   // 16 tokens x D/32 scale bytes of one page and head are contiguous
        if (lane < 2 * kScaleLanes)
          copy_async<16>(dst + s_dst, s_lane + static_cast<unsigned long long>(page) * s_stride + slot0 * (D / 32), page_ok);
      }
    } else {
#pragma unroll
      for (int x = 0; x < R::kCopies; ++x) {
        const int key = row_l + x * kStep;
        const long long row = key_row(key0 + key);
        const unsigned long long base = static_cast<unsigned long long>(row >= 0 ? row : 0) * stride;
        copy_async<16>(dst + key * R::kRow + R::place_k(key, piece) * 16, kp + base, row >= 0);
        copy_async<16>(dst + R::kOffV + key * R::kRow + R::place_v(key, piece) * 16, vp + base, row >= 0);
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

  auto begin = [&]() {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < count) issue(i);
      copy_commit();
    }
  };
  begin();
  if (F16 && __any_sync(0xffffffffu, tiny)) {
    bool lost = false;
#pragma unroll 1
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g8;
      const bool ok = r < row_count && (r0 + r) < rg.n * G;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(ok ? q_row(r) + c * (D / 4) : a.q);
      uint32_t top = 0;
#pragma unroll 1
      for (int i = 0; i < D / 4; ++i) top = max(top, src[i] & 0x7fffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
#pragma unroll 1
      for (int i = 0; i < D / 4; ++i) {
        const uint32_t x = src[i] & 0x7fffu;
        lost = lost || (ok && top < 0x7f80u && x != 0 && (x >> 7) + 31 < (top >> 7));
      }
    }
    if (__any_sync(0xffffffffu, lost)) {
      copy_wait<0>();
      __syncwarp();
      return false;
    }
  }
  while (true) {
    for (int i = 0; i < count; ++i) {
      copy_wait<kStages - 2>();
      __syncwarp();    // this stage has arrived for every lane; the stage before it has been read by every lane
      if (i + kStages - 1 < count) issue(i + kStages - 1);
      copy_commit();
      const uint8_t* st = ring + get * R::kStage;
      get = get + 1 == kStages ? 0 : get + 1;
      const int key0 = (t0 + i) * kTile;
      const int page_info = P16 ? 0 : *reinterpret_cast<const int*>(st + R::kOffPage);
      const bool tile_ok = P16 ? ((bad_tiles >> i) & 1) == 0 : page_info == 0xffff;
      const bool edge = key0 < all_lo || key0 + kTile > all_hi || !tile_ok;
      auto key_ok = [&](int k) {   // key0 + k holds a key of the cache that some row may see
        return key0 + k >= rg.lo && key0 + k < rg.hi && (P16 ? tile_ok : ((page_info >> k) & 1) != 0);
      };

      // ---- S^T = K Q^T
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
      float s2[NT][4];   // two chains of products, added at the end
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s2[nt][0] = s2[nt][1] = s2[nt][2] = s2[nt][3] = 0.0f;
      // Factors of this lane's share of keys g8, g8 + 8 and of value rows (2c, 2c + 1), (2c + 8, 2c + 9); for bf16 in two steps.
      uint32_t f1[2], g1[2], f2[2], g2[2];
      if constexpr (MX) {
        const uint8_t* sk = st + R::kOffS + g8 * (D / 32) + c * (D / 4) / 32;
        const uint8_t* sw = st + R::kOffS + R::kScale + 2 * c * (D / 32) + g8 * (D / 8) / 32;
        int bk[2] = {sk[0], sk[8 * (D / 32)]};
        int bv[4] = {sw[0], sw[D / 32], sw[8 * (D / 32)], sw[9 * (D / 32)]};
        if constexpr (F16) {
          // places above the lowest scale in reach: 0 .. kReach, or anything as unsigned numbers
          uint32_t uk[2], uv[4], most = 0;
#pragma unroll
          for (int j = 0; j < 2; ++j) uk[j] = bk[j] - (k_ref - kReach), most = max(most, uk[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) uv[j] = bv[j] - (v_ref - kReach), most = max(most, uv[j]);
          if (__any_sync(0xffffffffu, most > static_cast<uint32_t>(kReach))) {
            // rare: other references. NaN (255: the codes are NaN already) and keys that are none count for nothing
            int hk = kUnset, lk = 255, hv = kUnset, lv = 255;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (bk[j] == 255 || !key_ok(g8 + 8 * j)) bk[j] = -1;
              else hk = max(hk, bk[j]), lk = min(lk, bk[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (bv[j] == 255 || !key_ok(2 * c + (j & 1) + 8 * (j >> 1))) bv[j] = -1;
              else hv = max(hv, bv[j]), lv = min(lv, bv[j]);
            }
            hk = __reduce_max_sync(0xffffffffu, hk), lk = __reduce_min_sync(0xffffffffu, lk);
            hv = __reduce_max_sync(0xffffffffu, hv), lv = __reduce_min_sync(0xffffffffu, lv);
            hk = hk != kUnset ? hk : k_ref, hv = max(hv, v_ref);
            v_first = v_first != kUnset ? v_first : hv;
            if (lk < hk - kReach || lv < hv - kReach || hv - v_first > kClimb) {   // too far apart for f16
              copy_wait<0>();
              __syncwarp();
              return false;
            }
            k_ref = hk, k_unit = scale_value(k_ref);
            const float alpha = pow2_neg(v_ref - hv);
            v_ref = hv;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[d][nt][e] *= alpha;
#pragma unroll
            for (int j = 0; j < 2; ++j) uk[j] = bk[j] < 0 ? kReach : bk[j] - (k_ref - kReach);
#pragma unroll
            for (int j = 0; j < 4; ++j) uv[j] = bv[j] < 0 ? kReach : bv[j] - (v_ref - kReach);
          }
          // 2^(u - kReach) as f16: the exponent field is u + 1
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            f1[j] = uk[j] * 0x04000400u + 0x04000400u;
            g1[j] = uv[2 * j] * 0x400u + uv[2 * j + 1] * 0x04000000u + 0x04000400u;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int k0 = 2 * c + 8 * j;
            const uint32_t b = key_ok(g8 + 8 * j) ? bk[j] : 127, b0 = key_ok(k0) ? bv[2 * j] : 127, b1 = key_ok(k0 + 1) ? bv[2 * j + 1] : 127;
            f1[j] = mx_factor_first(b) * 0x10001u, f2[j] = mx_factor_second(b) * 0x10001u;
            g1[j] = mx_factor_first(b0) | mx_factor_first(b1) << 16, g2[j] = mx_factor_second(b0) | mx_factor_second(b1) << 16;
          }
        }
      }
      // four codes -> two registers of an operand, scaled
      auto scaled = [&](uint32_t w, uint32_t first, uint32_t second, uint32_t& lo, uint32_t& hi) {
        if constexpr (F16) {
          lo = mul_f16x2(codes_lo(w), first), hi = mul_f16x2(codes_hi(w), first);
        } else {
          mx_spread(w, lo, hi);
          lo = mul_bf16x2(mul_bf16x2(lo, first), second), hi = mul_bf16x2(mul_bf16x2(hi, first), second);
        }
      };
#pragma unroll
      for (int x = 0; x < R::kRow / 64; ++x) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(st + k_at[x]);
        const uint4 w1 = *reinterpret_cast<const uint4*>(st + k_at[x] + 8 * R::kRow);
        const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
        if constexpr (MX) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t fa[4];
            scaled(u0[y], f1[0], f2[0], fa[0], fa[2]);
            scaled(u1[y], f1[1], f2[1], fa[1], fa[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<F16>(y & 1 ? s2[nt] : s[nt], fa, qf[nt][2 * (4 * x + y)], qf[nt][2 * (4 * x + y) + 1]);
          }
        } else {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t fa[4] = {u0[2 * y], u1[2 * y], u0[2 * y + 1], u1[2 * y + 1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<false>(y & 1 ? s2[nt] : s[nt], fa, qf[nt][2 * (2 * x + y)], qf[nt][2 * (2 * x + y) + 1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = (s[nt][e] + s2[nt][e]) * (F16 ? factor[nt][e & 1] * k_unit : factor[nt][e & 1]);

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
        for (int e = 0; e < 4; ++e) raise = raise || s[nt][e] - m[nt][e & 1] > kRaise;
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(m[nt][e], fmaxf(s[nt][e], s[nt][e + 2]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float alpha = fast_exp2(m[nt][e] - mx);
            m[nt][e] = mx;
            l[nt][e] *= alpha, l[nt][e + 2] *= alpha;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) acc[d][nt][e] *= alpha, acc[d][nt][e + 2] *= alpha;
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // f16 probabilities are taken 2^7 times too large (below 2^15): small ones keep their bits; the sums carry the factor too,
        // and so do those of runs in bf16, which are joined with them
        const float c0 = m[nt][0] - (MX ? 7.0f : 0.0f), c1 = m[nt][1] - (MX ? 7.0f : 0.0f);
        const float p0 = fast_exp2(s[nt][0] - c0), p1 = fast_exp2(s[nt][1] - c1);
        const float p2 = fast_exp2(s[nt][2] - c0), p3 = fast_exp2(s[nt][3] - c1);
        pf[nt][0] = transpose_8x8(F16 ? pack_f16(p0, p1) : pack_bf16(p0, p1));
        pf[nt][1] = transpose_8x8(F16 ? pack_f16(p2, p3) : pack_bf16(p2, p3));
        constexpr uint32_t kOne = F16 ? 0x3c003c00u : 0x3f803f80u;
        const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
        mma_16816<F16>(l[nt], ones, pf[nt][0], pf[nt][1]);
      }

      // ---- O^T += V^T P^T: keys 2c, 2c + 1 (low, high half of a register) and 2c + 8, 2c + 9
      if constexpr (MX) {
        constexpr int kWords = R::kRow / 32;
        uint32_t v[4][kWords];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kWords == 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(st + v_at[0] + ((j & 1) + 8 * (j >> 1)) * R::kRow);
            v[j][0] = w.x, v[j][1] = w.y, v[j][2] = w.z, v[j][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(st + v_at[0] + ((j & 1) + 8 * (j >> 1)) * R::kRow);
            v[j][0] = w.x, v[j][1] = w.y;
          }
        }
#pragma unroll
        for (int y = 0; y < kWords; ++y) {
          uint32_t f[2][4];   // [key pair][channel 4y + .], each (first key, second key)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t ab = __byte_perm(v[2 * j][y], v[2 * j + 1][y], 0x5140), cd = __byte_perm(v[2 * j][y], v[2 * j + 1][y], 0x7362);
            scaled(ab, g1[j], g2[j], f[j][0], f[j][1]);
            scaled(cd, g1[j], g2[j], f[j][2], f[j][3]);
          }
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t fa[4] = {f[0][2 * z], f[0][2 * z + 1], f[1][2 * z], f[1][2 * z + 1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<F16>(acc[2 * y + z][nt], fa, pf[nt][0], pf[nt][1]);
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < R::kRow / 128; ++x) {
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(st + v_at[x] + ((j & 1) + 8 * (j >> 1)) * R::kRow);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t v0 = (&w[0].x)[y], v1 = (&w[1].x)[y], v2 = (&w[2].x)[y], v3 = (&w[3].x)[y];
            const uint32_t fa[4] = {__byte_perm(v0, v1, 0x5410), __byte_perm(v0, v1, 0x7632), __byte_perm(v2, v3, 0x5410),
                                    __byte_perm(v2, v3, 0x7632)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<false>(acc[4 * x + y][nt], fa, pf[nt][0], pf[nt][1]);
          }
        }
      }
    }
    left -= count;
    if (left <= 0) break;
    copy_wait<0>();
    __syncwarp();
    t0 += count, count = min(left, kPart / kTile);
    if constexpr (P16) look_up();
    begin();
  }
  copy_wait<0>();

  // ---- the run's result: rows 2c, 2c + 1 of every eight, channels g8 * D/8 + x
  const bool whole = rg.tiles <= split_tiles;   // no other run has keys: the result is final
  const float unit = F16 ? scale_value(v_ref) : 1.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * c + e;
      if (r >= row_count) continue;
      const float sum = l[nt][e];
      float f[D / 8];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) f[2 * d] = acc[d][nt][e] * unit, f[2 * d + 1] = acc[d][nt][e + 2] * unit;
      if (whole) {
        const int t = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
        // rows behind the sequence's last new token, and rows that see nothing, are zero
        const bool zero = (r0 + r) >= rg.n * G || sum == 0.0f;
        const float inv = 1.0f / sum;
        __nv_bfloat16* dst = a.out + ((static_cast<long long>(b) * a.T + t) * a.H + h) * D + g8 * (D / 8);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          uint32_t w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) w[y] = zero ? 0u : pack_bf16(f[8 * x + 2 * y] * inv, f[8 * x + 2 * y + 1] * inv);
          *reinterpret_cast<uint4*>(dst + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
        const long long at = (static_cast<long long>(b) * gridDim.y + blockIdx.y) * a.splits + split;
        const int rw = min(ROWS, a.T * G);
        float4* dst = reinterpret_cast<float4*>(a.part_o + (at * rw + r) * D + g8 * (D / 8));
#pragma unroll
        for (int x = 0; x < D / 32; ++x) dst[x] = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
        if (g8 == 0) *reinterpret_cast<float2*>(a.part_ml + (at * rw + r) * 2) = make_float2(m[nt][e], sum);
      }
    }
  return true;
}

// A function of its own, so that what f16 cannot hold takes no registers from what it can.
template <int D, int NT, bool P16>
__device__ __noinline__ void walk_in_bf16(const PagedAttnArgs& a, uint8_t* smem) {
  walk<D, true, false, NT, P16>(a, smem);
}

template <int D, bool MX, int NT, bool P16>
__global__ void __launch_bounds__(32, NT > 1 ? 8 : MX ? 16 : 12) paged_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  NC_PDL_PROLOGUE();
  if (!walk<D, MX, MX, NT, P16>(a, smem)) {
    if constexpr (MX) walk_in_bf16<D, NT, P16>(a, smem);
  }
}

// Rows per CTA: the query rows of a kv head in blocks of 8, 16 or 32.
int row_tiles(const PagedAttnArgs& a) {
  const int rows = a.T * (a.H / a.KV);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}

template <int D, bool MX, int NT, bool P16>
cudaError_t launch_rows(const PagedAttnArgs& a, cudaStream_t s) {
  using R = Ring<D, MX>;
  constexpr int ROWS = 8 * NT;
  static std::atomic<unsigned long long> configured{0};   // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if ((configured.load(std::memory_order_relaxed) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<D, MX, NT, P16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               R::kBytes);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit);
  }
  const int G = a.H / a.KV, blocks = (a.T * G + ROWS - 1) / ROWS;
  cudaError_t e = launch_maybe_pdl(paged_rows_kernel<D, MX, NT, P16>, dim3(a.splits, a.KV * blocks, a.B), dim3(32), R::kBytes, s, a);
  if (e != cudaSuccess || a.splits <= 1) return e;
  // always behind the first kernel's tail (it waits for it before it reads anything)
  return launch_combine<D>(a, ROWS, kTile, 1.0f, s);
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

bool paged_rows_can(const PagedAttnArgs& a) {
  const int G = a.H / a.KV, rows = 8 * row_tiles(a);
  return static_cast<long long>(a.KV) * ((static_cast<long long>(a.T) * G + rows - 1) / rows) <= 65535;
}

PagedPlan paged_rows_plan(const PagedAttnArgs& a) {
  const int G = a.H / a.KV, rows = 8 * row_tiles(a), blocks = (a.T * G + rows - 1) / rows;
  long long keys = std::min(static_cast<long long>(a.max_pages) * a.page_size, (1LL << 31) - kTile);   // lengths are ints
  if (a.window_left >= 0) keys = std::min(keys, static_cast<long long>(a.window_left) + 1 + (rows + G - 1) / G);
  const long long units = static_cast<long long>(a.B) * a.KV * blocks;
  // Runs that fill the warps of two CTAs per SM about three times over (so that the last ones even out), of 64 keys at
  // least (below that the fixed cost of a run and of joining it outweighs the keys) and 512 at most, unless that makes more than
  // twice as many: the runs, and with them the workspace (32 rows of D + 2 numbers each at most), are bounded. Units that
  // are enough by themselves are not split.
  const long long want = 148LL * 16 * 3;
  const auto share = [&](long long runs) { return static_cast<long long>(std::ceil(static_cast<double>(keys) * units / runs)); };
  long long per = std::max(std::min<long long>(std::max<long long>(share(want), 64), 512), share(2 * want));
  if (units >= want) per = keys + 2 * kTile;   // (a window may touch one tile more)
  per = (std::min<long long>(std::max<long long>(per, kTile), 1 << 30) + kTile - 1) / kTile * kTile;
  PagedPlan p;
  p.split_keys = static_cast<int>(per);
  // a window may start inside a tile and touch one more
  p.splits = static_cast<int>(((keys + kTile - 1) / kTile + (a.window_left >= 0 ? 1 : 0) + per / kTile - 1) / (per / kTile));
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
