// Shared by the two attention kernels over the paged cache (paged_rows.cu, paged_chunk.cu): which keys a block of rows
// sees, and the kernel that joins the partial results of rows whose keys were split.
//
// Rows: row r of a kv head of a sequence is query token r / G, head r % G of its group, G = H / KV. Runs of keys:
// run s of a block of rows covers `split_keys` keys from the block's first tile on.
#pragma once
#include <cuda_bf16.h>
#include <math_constants.h>

#include <algorithm>

#include "host_build.h"
#include "pdl_launch.h"
#include "ptx.cuh"
#include "serving.h"

namespace nc {

namespace {

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the rows [r0, r0 + rows) of sequence b see: row r is query token r / G, head r % G of the kv head's group.
struct Range {
  int n;             // new tokens of the sequence
  int base;          // position of its first new token
  int pmin, pmax;    // positions of the block's first and last real row
  int lo, hi;        // keys [lo, hi) that some row sees; hi <= lo: none
  int tile0, tiles;  // tiles of `tile` keys that cover them
};
__device__ __forceinline__ Range range_of(const PagedAttnArgs& a, int b, int r0, int rows, int tile) {
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
  g.tile0 = g.lo / tile;
  g.tiles = (g.hi + tile - 1) / tile - g.tile0;
  return g;
}

// out = sum_s o_s 2^(unit (m_s - M)) / sum_s l_s 2^(unit (m_s - M)) over the runs of a row; rows that one run finished are skipped.
// WARPS warps share a row (many runs, few rows), or each of the CTA's four warps takes a row (WARPS = 1).
template <int D, int WARPS>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnArgs a, int rows, int tile, float unit) {
  constexpr int ROWS_HERE = 4 / WARPS;
  __shared__ float sm_o[4][D], sm_l[4], sm_m[4];
  NC_PDL_PROLOGUE();
  const int G = a.H / a.KV, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WARPS;
  const int per = a.T * G;
  const long long id = static_cast<long long>(blockIdx.x) * ROWS_HERE + warp / WARPS;
  const bool inside = id < static_cast<long long>(a.B) * a.KV * per;
  const int r = inside ? static_cast<int>(id % per) : 0;
  const int kvh = inside ? static_cast<int>(id / per % a.KV) : 0, b = inside ? static_cast<int>(id / per / a.KV) : 0;
  const int rb = r / rows;
  const Range rg = range_of(a, b, rb * rows, rows, tile);
  const int split_tiles = a.split_keys / tile;
  const bool split = inside && rg.tiles > split_tiles;
  if (WARPS > 1 && !split) return;
  const bool real = r < rg.n * G;   // a row behind the last new token is zero
  const int n = split && real ? (rg.tiles + split_tiles - 1) / split_tiles : 0;
  const int rw = min(rows, per);
  const long long blocks = static_cast<long long>(a.KV) * ((per + rows - 1) / rows);
  const long long at = ((static_cast<long long>(b) * blocks + static_cast<long long>(rb) * a.KV + kvh) * a.splits) * rw + (r - rb * rows);
  float mx = -CUDART_INF_F;
  for (int s = part * 32 + lane; s < n; s += WARPS * 32) mx = fmaxf(mx, a.part_ml[(at + static_cast<long long>(s) * rw) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if constexpr (WARPS > 1) {
    if (lane == 0) sm_m[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sm_m[w]);
  }
  constexpr int E = D / 32;
  float o[E], ls = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int s = part; s < n; s += WARPS) {
    const long long p = at + static_cast<long long>(s) * rw;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
    const float w = ml.y == 0.0f ? 0.0f : fast_exp2((ml.x - mx) * unit);   // a run that the row saw nothing of
    ls = fmaf(w, ml.y, ls);
    if constexpr (E == 4) {
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + p * D + lane * 4);
      o[0] = fmaf(w, x.x, o[0]), o[1] = fmaf(w, x.y, o[1]), o[2] = fmaf(w, x.z, o[2]), o[3] = fmaf(w, x.w, o[3]);
    } else {
      const float2 x = *reinterpret_cast<const float2*>(a.part_o + p * D + lane * 2);
      o[0] = fmaf(w, x.x, o[0]), o[1] = fmaf(w, x.y, o[1]);
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sm_o[warp][lane * E + e] = o[e];
    if (lane == 0) sm_l[warp] = ls;
    __syncthreads();
    if (warp != 0) return;
    ls = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) ls += sm_l[w];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) o[e] += sm_o[w][lane * E + e];
    }
  }
  if (!split) return;
  const float inv = real && ls != 0.0f ? 1.0f / ls : 0.0f;
  __nv_bfloat16* dst = a.out + ((static_cast<long long>(b) * a.T + r / G) * a.H + kvh * G + r % G) * D;
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst + lane * 2) = pack_bf16(o[0] * inv, o[1] * inv);
}

// Always launched behind the first kernel's tail (it waits for that kernel before it reads anything).
template <int D>
cudaError_t launch_combine(const PagedAttnArgs& a, int rows, int tile, float unit, cudaStream_t s) {
  const long long total = static_cast<long long>(a.B) * a.T * a.H;
  if (total <= 2048)   // few rows: more loads in flight for each
    return launch_pdl(true, paged_combine_kernel<D, 4>, dim3(static_cast<unsigned>(total)), dim3(128), 0, s, a, rows, tile, unit);
  return launch_pdl(true, paged_combine_kernel<D, 1>, dim3(static_cast<unsigned>((total + 3) / 4)), dim3(128), 0, s, a, rows, tile, unit);
}

}  // namespace

}  // namespace nc
