// Attention of a chunk of new tokens over the paged cache (bf16 or MXFP8 pages): many rows per kv head, on tcgen05.
//
// Rows are (query token, head of the group): the heads that share a kv head are packed into the 128-row tiles of one CTA
// (the largest power of two that divides the group), so keys and values are read once for all of them and a chunk
// of a few tokens still fills a tile. A CTA takes two such tiles and walks the keys that either sees, 128 at a time:
//   warps 0..7, 8..15 softmax of row tile 0 and 1: two threads share a row, 64 keys each (one thread per row left a
//                     scheduler with one warp to issue from); P replaces S in tensor memory as bf16
//   warp 16           tcgen05.mma: S^x = Q^x K^T, O^x += P^x V, both in tensor memory all along
//   warp 17           TMA: Q; on bf16 pages also K and V, one 16-token box per page and 64 channels
//   warps 18..21 (K), 22..25 (V)  on MXFP8 pages: codes are copied (cp.async) one tile ahead, spread to bf16, multiplied by their
//                     block's power of two (exact) and stored in the operands' 128-byte swizzled layout
// The products run in the order O0(j), S0(j + 1), O1(j), S1(j + 1): while one tile's softmax works, the other tile's
// products do, and S(j + 1) needs no barrier of its own, because it follows the product that read P(j) out of its columns.
// 128 keys at a time because a 128 x 64 product from shared memory takes 48 clocks for the 32 of its arithmetic (the
// 128 rows of Q are read for every 64 keys), a 128 x 128 one the 64 it needs; and the waits of a step cost about 600.
// A page that is not in the pool, and 16 tokens that no row sees, become rows of zeros; values of the first and last
// 16 tokens that are only partly seen are copied by hand with zeros in the unseen places, because what lies there
// (a place behind the sequence's end) may be NaN, and 0 * NaN is not 0.
// The running maximum is raised only when a tile exceeds it by more than 2^8: then the thread rescales its O row in tensor
// memory. Bounds, per 128 x 128 tile: 1024 clocks for the exponentials (16 a clock and SM), 1024 for the two products.
// Probabilities are rounded to bf16, the tensor core's operand type of V's range; the row's sum takes them unrounded, in fp32 (each
// probability is off by 2^-8 of itself at most, in either direction).
// Measured (B200, D = 128): 2 x 2048 over 18k keys 387 us on bf16 pages (865 TFLOP/s), 482 on MXFP8 (694); 8 ragged
// prompts up to 2048, window 1024, 93 us.
// grid: (blocks of 256 rows x key runs, kv heads x head packs, sequences), the blocks that see most first.
#include <cuda.h>
#include <cuda_bf16.h>
#include <math_constants.h>

#include <atomic>

#include "mx_cache.cuh"
#include "paged_common.cuh"
#include "ptx.cuh"
#include "serving.h"
#include "tmap.h"

namespace nc {

namespace {

constexpr int BQ = 128;    // rows per tile (TMEM lanes)
constexpr int NQ = 2;      // row tiles per CTA
constexpr int kSoft = 8;   // softmax warps per row tile
constexpr int BKV = 128;   // keys per step
constexpr int KVS = 2;     // stages of K and of V
constexpr int kBox = 16;   // tokens per TMA box: a page holds a multiple of it
constexpr float kRescaleThreshold = 8.0f;  // log2 units

// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int D, bool MX>
struct ChunkLayout {
  static constexpr int kQ = BQ * D * 2;
  static constexpr int kKV = BKV * D * 2;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + NQ * kQ;
  static constexpr int kOffV = kOffK + KVS * kKV;
  static constexpr int kRaw = MX ? BKV * D : 0;                // codes of a tile, one side, as they lie in memory
  static constexpr int kOffRaw = kOffV + KVS * kKV;            // K, V
  static constexpr int kOffScale = kOffRaw + 2 * kRaw;         // scale bytes [BKV][D / 32], K, V
  static constexpr int kOffRow = kOffScale + (MX ? 2 * BKV * (D / 32) : 0);   // fp32 [NQ][BQ]: between a row's two threads
  static constexpr int kOffBar = kOffRow + NQ * BQ * 4;
  static constexpr int kTotal = kOffBar + 256;
  static_assert(kTotal <= 227 * 1024, "shared memory of one CTA");
  static constexpr int kThreads = (NQ * kSoft + 2 + (MX ? 8 : 0)) * 32;
};

struct ChunkParams {
  PagedAttnArgs a;   // a.KV counts packs of heads, a.H / a.KV heads each
  int kv_per_pack;   // real kv head = pack / kv_per_pack
  int KV;            // real kv heads
};

template <int D, bool MX>
__global__ void __launch_bounds__(ChunkLayout<D, MX>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const ChunkParams p) {
  using L = ChunkLayout<D, MX>;
  constexpr int DC = D / 64;
  const PagedAttnArgs& a = p.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023) != 0) {   // the operands' swizzle wants it; there is no room to align by hand
    if (threadIdx.x == 0 && a.status != nullptr) atomicCAS(a.status, 0, kErrWaitOther);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + KVS;
  uint64_t* v_full = k_empty + KVS;
  uint64_t* v_empty = v_full + KVS;
  uint64_t* s_full = v_empty + KVS;      // [NQ] scores of a key tile are there
  uint64_t* p_full = s_full + NQ;        // [NQ] its probabilities are, in their place
  uint64_t* o_final = p_full + NQ;       // [NQ] the last P V product is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_final + NQ);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.KV;                               // heads in a pack: a power of two
  const int blocks = (a.T * G + NQ * BQ - 1) / (NQ * BQ);
  const int qb = blocks - 1 - static_cast<int>(blockIdx.x) / a.splits, split = blockIdx.x % a.splits;
  const int pack = blockIdx.y, kvh = pack / p.kv_per_pack, b = blockIdx.z;
  const int r0 = qb * NQ * BQ, row_count = min(NQ * BQ, a.T * G - r0);
  const Range rg = range_of(a, b, r0, NQ * BQ, BKV);
  const int split_tiles = a.split_keys / BKV;
  const bool whole = rg.tiles <= split_tiles;             // no other run has keys: the result is final
  const int first = rg.tile0 + split * split_tiles;
  const int n_u = min(rg.tiles - split * split_tiles, split_tiles);   // key tiles of this CTA
  if (split > 0 && n_u <= 0) return;
  if (split == 0 && threadIdx.x == 0 && rg.pmax >= static_cast<long long>(a.max_pages) * a.page_size && a.status != nullptr)
    atomicCAS(a.status, 0, kErrBadIndex);   // keys past the page table are left out
  auto out_row = [&](int r) {   // row r of the block
    return a.out + ((static_cast<long long>(b) * a.T + (r0 + r) / G) * a.H + pack * G + (r0 + r) % G) * D;
  };
  if (n_u <= 0) {               // nothing is seen: zeros
    for (int i = threadIdx.x; i < row_count * (D / 8); i += L::kThreads)
      reinterpret_cast<uint4*>(out_row(i / (D / 8)))[i % (D / 8)] = make_uint4(0, 0, 0, 0);
    return;
  }
  // key tiles of each row tile inside this CTA's run
  int lo[NQ], hi[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const Range t = range_of(a, b, r0 + x * BQ, BQ, BKV);
    lo[x] = max(t.tile0, first);
    hi[x] = t.tiles > 0 ? min(t.tile0 + t.tiles - 1, first + n_u - 1) : -1;
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < KVS; ++i) {
      mbar_init(&k_full[i], MX ? 4 : 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], MX ? 4 : 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int x = 0; x < NQ; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], kSoft);
      mbar_init(&o_final[x], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == NQ * kSoft) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  const int* table = a.page_table + static_cast<long long>(b) * a.max_pages;
  // A page that is none of the pool's is found here once; only then are pages looked at again where scores are masked.
  bool bad = false;
  for (int pg = max(first * BKV, rg.lo) / a.page_size + threadIdx.x; pg <= (min((first + n_u) * BKV, rg.hi) - 1) / a.page_size;
       pg += L::kThreads) {
    const int page = table[pg];
    bad = bad || page < 0 || page >= a.num_pages;
  }
  if (bad && a.status != nullptr) atomicCAS(a.status, 0, kErrBadIndex);
  tc_fence_before();
  const bool any_bad = __syncthreads_or(bad);
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto tmem_S = [&](int x) { return tmem_base + x * BKV; };
  auto tmem_O = [&](int x) { return tmem_base + 256 + x * 128; };

  if (warp == NQ * kSoft) {
    // ---------------------------------------------------------------- MMA issuer
    // The whole warp walks the loop and waits, one elected thread issues: control flow and descriptors stay uniform
    // (a single lane that ran it alone took 44 clocks to issue a product).
    constexpr uint32_t idesc_s = make_idesc_bf16(BQ, BKV, false, false);
    constexpr uint32_t idesc_o = make_idesc_bf16(BQ, D, false, true);
    const uint64_t q_desc0 = make_smem_desc_sw128(smem_u32(smem + L::kOffQ), 16, 1024);
    const uint64_t k_desc0 = make_smem_desc_sw128(smem_u32(smem + L::kOffK), 16, 1024);
    const uint64_t v_desc0 = make_smem_desc_sw128(smem_u32(smem + L::kOffV), BKV * 128, 1024);
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, code)) != 0;
    };
    auto sees = [&](int x, int j) { return j >= lo[x] && j <= hi[x]; };
    auto scores = [&](int x, int s) {          // S^x of key tile first + s
      const uint64_t dq = q_desc0 + static_cast<uint64_t>(x * (L::kQ >> 4));
      const uint64_t dk = k_desc0 + static_cast<uint64_t>((s % KVS) * (L::kKV >> 4));
      const uint32_t ts = tmem_S(x);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t qo = static_cast<uint64_t>(((k / 4) * (BQ * 128) + (k % 4) * 32) >> 4);
          const uint64_t ko = static_cast<uint64_t>(((k / 4) * (BKV * 128) + (k % 4) * 32) >> 4);
          mma_f16_ss(ts, dq + qo, dk + ko, idesc_s, k > 0 ? 1u : 0u);
        }
        mma_commit(&s_full[x]);
      }
      __syncwarp();
    };
    auto free_stage = [&](uint64_t* bar) {
      if (elect_one()) mma_commit(bar);
      __syncwarp();
    };
    bool ok = wait(q_full, 0, kErrWaitFull) && wait(&k_full[0], 0, kErrWaitFull);
    if (ok) {
      tc_fence_after();
      for (int x = 0; x < NQ; ++x)
        if (sees(x, first)) scores(x, 0);
      free_stage(&k_empty[0]);
    }
    for (int s = 0; s < n_u && ok; ++s) {
      const int j = first + s, st = s % KVS;
      bool have_v = false, have_k = false;
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        if (ok && sees(x, j)) {
          if (!have_v) ok = wait(&v_full[st], (s / KVS) & 1, kErrWaitFull), have_v = true;
          ok = ok && wait(&p_full[x], (j - lo[x]) & 1, kErrWaitOther);
          if (ok) {
            tc_fence_after();
            const uint64_t dv = v_desc0 + static_cast<uint64_t>(st * (L::kKV >> 4));
            const uint32_t ts = tmem_S(x), to = tmem_O(x);
            const uint32_t more = j > lo[x] ? 1u : 0u;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < BKV / 16; ++k)   // P of 64 keys takes the first 32 of their 64 score columns
                mma_f16_ts(to, ts + (k / 4) * 64 + (k % 4) * 8, dv + static_cast<uint64_t>((k * 16 * 128) >> 4), idesc_o,
                           k > 0 ? 1u : more);
              if (j == hi[x]) mma_commit(&o_final[x]);
            }
            __syncwarp();
          }
        }
        if (ok && s + 1 < n_u && sees(x, j + 1)) {
          if (!have_k) ok = wait(&k_full[(s + 1) % KVS], ((s + 1) / KVS) & 1, kErrWaitFull), have_k = true;
          if (ok) {
            tc_fence_after();
            scores(x, s + 1);
          }
        }
      }
      if (ok) {
        if (!have_v) ok = wait(&v_full[st], (s / KVS) & 1, kErrWaitFull);   // a tile that neither row tile sees
        if (ok && s + 1 < n_u && !have_k) ok = wait(&k_full[(s + 1) % KVS], ((s + 1) / KVS) & 1, kErrWaitFull);
        if (ok) {
          free_stage(&v_empty[st]);
          if (s + 1 < n_u) free_stage(&k_empty[(s + 1) % KVS]);
        }
      }
    }
  } else if (warp == NQ * kSoft + 1) {
    // ---------------------------------------------------------------- TMA: Q, and bf16 keys and values
    if (lane == 0) {
      mbar_expect_tx(q_full, NQ * L::kQ);
#pragma unroll
      for (int x = 0; x < NQ; ++x)
#pragma unroll
        for (int c = 0; c < DC; ++c)   // tokens past T are read as zeros
          tma_load_4d(smem + L::kOffQ + x * L::kQ + c * (BQ * 128), &tmQ, q_full, c * 64, pack * G, (r0 + x * BQ) / G, b);
    }
    bool ok = true;
    if constexpr (!MX) {
      const int out_of_pool = a.num_pages * a.page_size;   // a row outside the map: the box arrives as zeros
      int st = 0;
      uint32_t ph = 0;
      for (int s = 0; s < n_u && ok; ++s) {
        // lanes 0..7: the boxes of the tile
        const int key = (first + s) * BKV + (lane & 7) * kBox;
        int row = out_of_pool;
        bool partial = false;
        if (key + kBox > rg.lo && key < rg.hi) {
          const int page = table[key / a.page_size];
          if (page >= 0 && page < a.num_pages) row = page * a.page_size + key % a.page_size;
          partial = row != out_of_pool && (key < rg.lo || key + kBox > rg.hi);
        }
        const unsigned by_hand = __ballot_sync(0xffffffffu, partial && lane < BKV / kBox);
        ok = mbar_wait(&k_empty[st], ph ^ 1, abort_flag, a.status, kErrWaitEmpty);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        uint8_t* sk = smem + L::kOffK + st * L::kKV;
        uint8_t* sv = smem + L::kOffV + st * L::kKV;
        if (lane == 0) mbar_expect_tx(&k_full[st], L::kKV);
        __syncwarp();
        if (lane < BKV / kBox)
#pragma unroll
          for (int c = 0; c < DC; ++c)
            tma_load_3d(sk + c * (BKV * 128) + lane * (kBox * 128), &tmK, &k_full[st], c * 64, row, kvh);
        __syncwarp();
        ok = mbar_wait(&v_empty[st], ph ^ 1, abort_flag, a.status, kErrWaitEmpty);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (by_hand != 0) {
          for (int box = 0; box < BKV / kBox; ++box) {
            if (((by_hand >> box) & 1) == 0) continue;
            const int row_b = __shfl_sync(0xffffffffu, row, box), key_b = (first + s) * BKV + box * kBox;
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.v_pool) +
                                       (static_cast<long long>(row_b) * p.KV + kvh) * D;
            for (int i = lane; i < kBox * (D / 8); i += 32) {
              const int t = i / (D / 8), u = i % (D / 8);
              uint4 w = make_uint4(0, 0, 0, 0);
              if (key_b + t >= rg.lo && key_b + t < rg.hi)
                w = *reinterpret_cast<const uint4*>(src + static_cast<long long>(t) * p.KV * D + u * 8);
              *reinterpret_cast<uint4*>(sv + (u >> 3) * (BKV * 128) + (box * kBox + t) * 128 + (((u & 7) ^ (t & 7)) * 16)) = w;
            }
          }
          fence_async_shared();
          __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(&v_full[st], L::kKV - __popc(by_hand) * kBox * D * 2);
        __syncwarp();
        if (lane < BKV / kBox && !partial)
#pragma unroll
          for (int c = 0; c < DC; ++c)
            tma_load_3d(sv + c * (BKV * 128) + lane * (kBox * 128), &tmV, &v_full[st], c * 64, row, kvh);
        if (++st == KVS) { st = 0; ph ^= 1; }
      }
    }
    if (!ok) {   // copies in flight land before the CTA ends
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
  } else if (MX && warp >= NQ * kSoft + 2) {
    // ---------------------------------------------------------------- MXFP8 keys and values -> bf16 operands
    if constexpr (MX) {
      constexpr int U = D / 16;                 // 16-code pieces of a row
      constexpr int N = BKV * U / 128;          // pieces per thread and side: rows t / U + i * (128 / U)
      constexpr int kRows = 128 / U, kBoxStep = kRows / kBox;
      const int side = (warp - (NQ * kSoft + 2)) >> 2;   // 0: keys, 1: values
      const int t = (threadIdx.x - (NQ * kSoft + 2) * 32) & 127;
      const int row0 = t / U, u = t % U, in_box = row0 % kBox, box0 = row0 / kBox;
      const uint32_t stride = static_cast<uint32_t>(p.KV) * D, s_stride = static_cast<uint32_t>(p.KV) * a.page_size * (D / 32);
      const uint8_t* codes = static_cast<const uint8_t*>(side ? a.v_pool : a.k_pool) + static_cast<long long>(in_box) * stride + kvh * D + u * 16;
      const uint8_t* scales = (side ? a.v_scale : a.k_scale) + (static_cast<long long>(kvh) * a.page_size + in_box) * (D / 32);
      const uint32_t raw = smem_u32(smem + L::kOffRaw) + side * L::kRaw + t * 16;
      uint8_t* const scale_sm = smem + L::kOffScale + side * BKV * (D / 32);
      const uint32_t scale_at = smem_u32(scale_sm);
      uint64_t *full = side ? v_full : k_full, *empty = side ? v_empty : k_empty;
      // Lanes 0..7 look up the pages of a tile's eight boxes, two tiles ahead of its codes: the number is asked for here and
      // looked at in `settle`, a tile later. Slot of a box in its page: the same for all tiles but for the page's turn.
      int next_id = -1, next_slot = 0, page_l = -1, slot_l = 0;
      bool plain = false;   // every row of the tile is wanted and every page is one of the pool's
      auto look = [&](int s) {
        const int key = (first + s) * BKV + (lane & 7) * kBox;
        next_id = -1, next_slot = 0;
        if (s < n_u && key + kBox > rg.lo && key < rg.hi) {
          const int lp = key / a.page_size;
          next_slot = key - lp * a.page_size;
          next_id = table[lp];
        }
      };
      auto settle = [&](int s) {
        page_l = next_id >= 0 && next_id < a.num_pages ? next_id : -1, slot_l = next_slot;
        plain = (first + s) * BKV >= rg.lo && (first + s + 1) * BKV <= rg.hi && __all_sync(0xffffffffu, page_l >= 0);
      };
      // A thread copies the pieces that it will convert; rows and pages that are not wanted arrive as zeros. The scale bytes of
      // a row (or of two, where they are two each: a copy takes four) come with its first piece, for the whole warp.
      auto fetch = [&](int s) {
        if (s < n_u) {
#pragma unroll 4
          for (int i = 0; i < N; ++i) {
            const int box = box0 + i * kBoxStep, r = row0 + i * kRows, key = (first + s) * BKV + r;
            const int id = __shfl_sync(0xffffffffu, page_l, box), slot = __shfl_sync(0xffffffffu, slot_l, box);
            const bool ok = plain || (id >= 0 && key >= rg.lo && key < rg.hi);
            const bool two = D == 64 && (plain || (ok && key + 1 < rg.hi));
            const unsigned page = id >= 0 ? id : 0;
            const uint8_t* c = codes + static_cast<unsigned long long>(page * static_cast<unsigned>(a.page_size) + slot) * stride;
            const uint8_t* sc = scales + static_cast<unsigned long long>(page) * s_stride + slot * (D / 32);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw + i * 2048), "l"(c), "r"(ok ? 16 : 0) : "memory");
            if (u == 0 && (D == 128 || (r & 1) == 0))
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(scale_at + r * (D / 32)), "l"(sc),
                           "r"(D == 128 ? (ok ? 4 : 0) : (two || (id >= 0 && key + 1 >= rg.lo && key + 1 < rg.hi) ? 4 : ok ? 2 : 0))
                           : "memory");
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      auto store = [&](uint8_t* base) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < N; ++i) {
          const int r = row0 + i * kRows;
          uint4 code;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(code.x), "=r"(code.y), "=r"(code.z), "=r"(code.w)
                       : "r"(raw + i * 2048) : "memory");
          const uint32_t sb = scale_sm[r * (D / 32) + u / 2];
          const uint32_t f1 = mx_factor_first(sb) * 0x10001u;
          const uint32_t w[4] = {code.x, code.y, code.z, code.w};
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            mx_spread(w[y], o[2 * y], o[2 * y + 1]);
            o[2 * y] = mul_bf16x2(o[2 * y], f1), o[2 * y + 1] = mul_bf16x2(o[2 * y + 1], f1);
          }
          if (sb > 134u) {
            const uint32_t f2 = mx_factor_second(sb) * 0x10001u;
            const bool zero = (code.x | code.y | code.z | code.w) == 0;   // rows that are none, beside scales that may be anything
#pragma unroll
            for (int y = 0; y < 8; ++y) o[y] = zero ? 0u : mul_bf16x2(o[y], f2);
          }
          uint8_t* row = base + (u >> 2) * (BKV * 128) + r * 128;
          const int g = (u & 3) * 2;
          *reinterpret_cast<uint4*>(row + ((g ^ (r & 7)) * 16)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(row + (((g + 1) ^ (r & 7)) * 16)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_async_shared();
        __syncwarp();
      };
      int st = 0;
      uint32_t ph = 0;
      // the next codes are requested as soon as the staging area is free, and arrive while this warp waits for a stage
      look(0);
      settle(0);
      fetch(0);
      look(1);
      for (int s = 0; s < n_u; ++s) {
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[st], ph ^ 1, abort_flag, a.status, kErrWaitEmpty))) break;
        store(smem + (side ? L::kOffV : L::kOffK) + st * L::kKV);
        if (lane == 0) mbar_arrive(&full[st]);
        settle(s + 1);
        fetch(s + 1);
        look(s + 2);
        if (++st == KVS) { st = 0; ph ^= 1; }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int x = warp / kSoft, half = (warp >> 2) & 1;   // this thread's 64 of the 128 keys of a step
    const int row = (warp & 3) * 32 + lane;      // (a warp reaches the 32 TMEM lanes of its number modulo 4)
    const int pair_bar = 1 + x * 4 + (warp & 3);   // named barrier of the two warps that share 32 rows
    float* const row_max = reinterpret_cast<float*>(smem + L::kOffRow) + x * BQ + row;
    const int r = r0 + x * BQ + row;             // row of the pack
    const bool row_in = x * BQ + row < row_count, real = r < rg.n * G;
    const int qpos = real ? rg.base + r / G : -1;
    const int t_last = min((r0 + x * BQ + BQ - 1) / G, rg.n - 1);
    const int pos_min = rg.base + (r0 + x * BQ) / G, pos_max = rg.base + t_last;   // of the tile's real rows
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int n_x = hi[x] - lo[x] + 1;
    const float sl = a.scale * 1.4426950408889634f;
    float m_ref = -1.0e30f, l_run = 0.0f;
    bool ok = true;
    // Some row of the warp has a reference so large that rounding reference * sl would show (from 2^10 on by more than 2^-14 of a
    // probability, from 2^31 on by all of it): the reference is taken from the scores before they are scaled.
    bool far = false;
    float sv[32];
    for (int i = 0; i < n_x; ++i) {
      const int kv0 = (lo[x] + i) * BKV + half * 64;
      const bool need_mask = any_bad || kv0 + 63 > pos_min || (a.window_left >= 0 && kv0 < pos_max - a.window_left) || kv0 + 64 > rg.hi;
      // scores of 32 keys, unseen ones -infinity: the maximum wants all first, so one of the two pieces is read twice
      auto load = [&](int piece) {
        uint32_t rv[32];
        tmem_ld_32x32(tmem_S(x) + half * 64 + piece * 32 + lane_sel, rv);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) sv[e] = __uint_as_float(rv[e]);
        if (!need_mask) return;
        // keys [k_lo, k_hi) of the piece are seen by the row; the rest cannot be told from seen ones by value
        const int k0 = kv0 + piece * 32;
        const int k_hi = min(qpos + 1, rg.hi) - k0, k_lo = (a.window_left >= 0 ? max(0, qpos - a.window_left) : 0) - k0;
#pragma unroll
        for (int e = 0; e < 32; ++e) sv[e] = e >= k_lo && e < k_hi ? sv[e] : -CUDART_INF_F;
        for (int box = 0; any_bad && box < 32 / kBox; ++box) {   // a page outside the pool: its keys are none
          const int key = k0 + box * kBox;
          if (key >= rg.hi || key + kBox <= rg.lo) continue;
          const int page = table[key / a.page_size];
          if (page < 0 || page >= a.num_pages) {
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[e] = (e >> 4) == box ? -CUDART_INF_F : sv[e];
          }
        }
      };
      auto largest = [&](float m) {
        float mt[4] = {m, m, m, m};   // four chains, three operands an instruction
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int c = 0; c < 4; ++c) mt[c] = fmaxf(fmaxf(mt[c], sv[e + 2 * c]), sv[e + 2 * c + 1]);
        return fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3]));
      };
      auto probabilities = [&](int piece) {
        if (far) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) unpack2(add2(pack2(sv[e], sv[e + 1]), pack2(-m_ref, -m_ref)), sv[e], sv[e + 1]);
        }
        const float off = far ? 0.0f : -m_ref * sl;
        const uint64_t sl2 = pack2(sl, sl), m2 = pack2(off, off);
        uint32_t packed[16];
        uint64_t sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float p0, p1;
          unpack2(fma2(pack2(sv[e], sv[e + 1]), sl2, m2), p0, p1);
          p0 = fast_exp2(p0), p1 = fast_exp2(p1);
          sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pack2(p0, p1));
          packed[e / 2] = pack_bf16(p0, p1);
        }
        float l0, l1;
        unpack2(add2(sum[0], sum[1]), l0, l1);
        l_run += l0 + l1;
        tmem_st_32x16(tmem_S(x) + half * 64 + piece * 16 + lane_sel, packed);
      };
      // A wait that gives up leaves the loop's barriers in step: every thread of the tile goes on, on whatever there is.
      ok = mbar_wait(&s_full[x], i & 1, abort_flag, a.status, kErrWaitTmemFull) && ok;
      tc_fence_after();
      load(1);
      float m_tile = largest(-1.0e30f);
      load(0);
      m_tile = largest(m_tile);
      // Both threads of a row have to use one reference. Whether any of the pair's rows wants a higher one is a barrier
      // with a vote; only then the maxima themselves are exchanged, in fp32 (a reference above the true maximum by as little
      // as 2^-8 of it loses every probability of a row with large scores) through one word per row, which is all that
      // there is room for. The next vote keeps a next exchange behind this one's reads.
      const bool raise = (m_tile - m_ref) * sl > kRescaleThreshold;
      uint32_t any_raise;
      asm volatile(
          "{\n"
          ".reg .pred p, q;\n"
          "setp.ne.u32 p, %1, 0;\n"
          "bar.red.or.pred q, %2, 64, p;\n"
          "selp.u32 %0, 1, 0, q;\n"
          "}\n"
          : "=r"(any_raise)
          : "r"(static_cast<uint32_t>(raise)), "r"(pair_bar)
          : "memory");
      if (any_raise) {
        if (half == 1) *row_max = m_tile;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        if (half == 0) *row_max = m_tile = fmaxf(m_tile, *row_max);
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        if (half == 1) m_tile = *row_max;
        float alpha = 1.0f;
        if ((m_tile - m_ref) * sl > kRescaleThreshold) {
          alpha = fast_exp2((m_ref - m_tile) * sl);
          m_ref = m_tile;
          l_run *= alpha;
        }
        far = __any_sync(0xffffffffu, m_ref > -1.0e30f && fabsf(m_ref * sl) > 1024.0f);
        if (i > 0) {   // the scores of this tile came after the P V product of the one before: O is at rest
#pragma unroll 1
          for (int c = half * (D / 32); c < (half + 1) * (D / 32); ++c) {
            uint32_t o[16];
            tmem_ld_32x16(tmem_O(x) + c * 16 + lane_sel, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x16(tmem_O(x) + c * 16 + lane_sel, o);
          }
        }
      }
      probabilities(0);   // into the place of the first 16 of the 32 columns that are in registers
      load(1);
      probabilities(1);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x]);
    }
    if (ok && n_x > 0) ok = mbar_wait(&o_final[x], 0, abort_flag, a.status, kErrWaitTmemFull);
    const bool any = n_x > 0;                 // else O was never written
    if (any) {   // the row's sum: its halves meet where this tile's Q was, which no product reads any more
      float* const halves = reinterpret_cast<float*>(smem + L::kOffQ + x * L::kQ) + row;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      if (ok) halves[half * BQ] = l_run;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      if (ok) l_run += halves[(half ^ 1) * BQ];
    }
    if (ok) {
      tc_fence_after();
      if (whole) {
        const bool zero = !any || !real || l_run == 0.0f;
        const float inv_l = 1.0f / l_run;
        __nv_bfloat16* op = out_row(x * BQ + (row_in ? row : 0));
#pragma unroll 1
        for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
          uint32_t w[32];
          if (any) {
            tmem_ld_32x32(tmem_O(x) + c * 32 + lane_sel, w);
            tmem_ld_wait();
          }
          if (row_in) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] = zero ? 0u : pack_bf16(__uint_as_float(w[g * 8 + e * 2]) * inv_l, __uint_as_float(w[g * 8 + e * 2 + 1]) * inv_l);
              *reinterpret_cast<uint4*>(op + c * 32 + g * 8) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        }
      } else {
        const int rw = min(NQ * BQ, a.T * G);
        const long long at = ((static_cast<long long>(b) * gridDim.y * blocks + static_cast<long long>(qb) * gridDim.y + pack) *
                                  a.splits + split) * rw + x * BQ + row;
        float* dst = a.part_o + at * D;
#pragma unroll 1
        for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
          uint32_t w[32];
          if (any) {
            tmem_ld_32x32(tmem_O(x) + c * 32 + lane_sel, w);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = 0;
          }
          if (row_in) {
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<uint4*>(dst + c * 32 + g * 4) = make_uint4(w[g * 4], w[g * 4 + 1], w[g * 4 + 2], w[g * 4 + 3]);
          }
        }
        // (the reference before the scale: the difference of two is exact where their products with it are not)
        if (row_in && half == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_ref, any ? l_run : 0.0f);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == NQ * kSoft) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Heads per pack: the largest power of two (at most a tile) that divides the group.
int pack_of(int G) {
  int p = 1;
  while (p < BQ && G % (2 * p) == 0) p *= 2;
  return p;
}

template <int D, bool MX>
const char* launch_chunk(const PagedAttnArgs& args, cudaStream_t s) {
  using L = ChunkLayout<D, MX>;
  ChunkParams p;
  p.a = args;
  const int G = args.H / args.KV, P = pack_of(G);
  p.KV = args.KV;
  p.kv_per_pack = G / P;
  p.a.KV = args.H / P;
  CUtensorMap tq, tk, tv;
  const long long dq[4] = {D, args.H, args.T, args.B};
  const long long sq[3] = {args.q_stride_h, args.q_stride_t, args.q_stride_b};
  const int boxq[4] = {64, P, BQ / P, 1};
  if (!make_tmap_bf16_4d(&tq, args.q, dq, sq, boxq)) return "paged_chunk_attention: tensor map construction failed";
  tk = tv = tq;
  if (!MX) {
    const long long rows = static_cast<long long>(args.num_pages) * args.page_size, stride = static_cast<long long>(args.KV) * D;
    if (!make_tmap_bf16_3d(&tk, args.k_pool, D, rows, args.KV, stride, D, 64, kBox) ||
        !make_tmap_bf16_3d(&tv, args.v_pool, D, rows, args.KV, stride, D, 64, kBox))
      return "paged_chunk_attention: tensor map construction failed";
  }
  static std::atomic<unsigned long long> configured{0};   // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if ((configured.load(std::memory_order_relaxed) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(paged_chunk_kernel<D, MX>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal);
    if (e != cudaSuccess) return cudaGetErrorString(e);
    configured.fetch_or(bit);
  }
  const int blocks = (args.T * P + NQ * BQ - 1) / (NQ * BQ);
  const dim3 grid(static_cast<unsigned>(blocks) * args.splits, p.a.KV, args.B);
  paged_chunk_kernel<D, MX><<<grid, L::kThreads, L::kTotal, s>>>(tq, tk, tv, p);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && args.splits > 1) e = launch_combine<D>(p.a, NQ * BQ, BKV, args.scale * 1.4426950408889634f, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

PagedPlan paged_chunk_plan(const PagedAttnArgs& a) {
  const int P = pack_of(a.H / a.KV), rows = NQ * BQ, blocks = (a.T * P + rows - 1) / rows;
  long long keys = static_cast<long long>(a.max_pages) * a.page_size;
  if (a.window_left >= 0) keys = std::min(keys, static_cast<long long>(a.window_left) + 1 + rows / P);
  const long long units = static_cast<long long>(a.B) * (a.H / P) * blocks;
  // One CTA per SM: four waves of them, so that the last one is a small part; runs of 512 keys at least (joining a run
  // costs as much as some 100 keys).
  const long long want = (148 * 4 + units - 1) / units;
  long long per = ((keys + want - 1) / want + BKV - 1) / BKV * BKV;
  per = std::max<long long>(per, 512);
  PagedPlan p;
  p.split_keys = static_cast<int>(std::min<long long>(per, 1 << 30));
  // a window may start inside a tile and touch one more
  p.splits = static_cast<int>(((keys + BKV - 1) / BKV + (a.window_left >= 0 ? 1 : 0) + per / BKV - 1) / (per / BKV));
  if (want == 1) p.splits = 1, p.split_keys = 1 << 30;
  if (p.splits > 1) {
    const long long rw = std::min<long long>(rows, static_cast<long long>(a.T) * P);
    p.part_o = units * p.splits * rw * a.D;
    p.part_ml = units * p.splits * rw * 2;
  }
  return p;
}

bool paged_chunk_can(const PagedAttnArgs& a) {
  // TMA boxes are 16 tokens of one page. A scale that is not positive turns the maximum around.
  return a.page_size % kBox == 0 && a.scale > 0.0f && a.H / pack_of(a.H / a.KV) <= 65535 &&
         static_cast<long long>(a.num_pages) * a.page_size < (1LL << 31) - 1024;
}

bool paged_chunk_takes(const PagedAttnArgs& a) {
  // Few rows per kv head leave most of a 128-row tile empty, and the other kernel reads the keys at full speed: 16 sequences,
  // 4 kv heads, 4000 keys of 128 channels, other / this kernel: 16 rows 53 / 66 us (bf16 pages), 49 / 75 (MXFP8), 20 rows 83 / 68 and
  // 76 / 78, 32 rows 96 / 70 and 88 / 80. (Of 64 channels they meet between 32 and 64 rows: at 32, 49 / 59 and 57 / 68.)
  // Little work in all is done before this kernel has started up. The rule of 1.5 GFLOP, counted over the page table's width because a
  // captured call knows no lengths, is coarse: 3 x 77 tokens, 4 heads of 64: 777 keys (0.2 GFLOP) 19 / 25 us, 3077 keys (0.7) 31 / 26;
  // 1 x 200, 8 heads of 128: 200 keys (0.2) 23 / 16, 1000 keys (0.8) 27 / 31, 2200 keys (1.8) 49 / 31.
  double keys = static_cast<double>(a.max_pages) * a.page_size;
  if (a.window_left >= 0) keys = std::min(keys, static_cast<double>(a.window_left) + 1 + a.T);
  return a.T * (a.H / a.KV) > 16 && 4.0 * a.D * a.H * a.T * a.B * keys > 1.5e9 && paged_chunk_can(a);
}

const char* paged_chunk_attention(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.T == 0) return nullptr;
  if (a.splits > 1 && (a.part_o == nullptr || a.part_ml == nullptr)) return "paged attention: no workspace for the key splits";
  const bool mx = a.k_scale != nullptr;
  if (a.D == 128) return mx ? launch_chunk<128, true>(a, s) : launch_chunk<128, false>(a, s);
  return mx ? launch_chunk<64, true>(a, s) : launch_chunk<64, false>(a, s);
}

}  // namespace nc
