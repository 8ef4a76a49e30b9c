// The MXFP8 key / value cache: rows are quantised as they are written into their pages, and read back as bf16.
//
// A block is 32 channels of one token and head: code = e4m3(x * 2^(127 - b)), value = code * 2^(b - 127) with b from the
// block's largest magnitude (mx_cache.cuh). Scales being powers of two, scaling is exact in both directions and the code
// is the only rounding. Both kernels only move bytes (append: 2 read, 1 + 1/32 written per element; read: the reverse),
// so what counts is that a thread has all its loads in flight at once and that every access is 16 bytes wide: a
// thread owns 16 channels of one row, two threads share a block and exchange their maxima by one shuffle.
// The scale pool is laid out [page, head, token, block]: the scales of one page and head, which the attention
// kernels read together, are contiguous.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host_build.h"
#include "mx_cache.cuh"
#include "mx_quant.cuh"
#include "pdl_launch.h"
#include "ptx.cuh"
#include "serving.h"

namespace nc {

namespace {

constexpr int kThreads = 256;

// Where the row of (token, head) lives; false: not a usable place (a negative position is simply not one).
__device__ __forceinline__ bool place(const MxCache& c, int b, int pos, int h, int* status, bool report, long long& row,
                                      long long& srow) {
  if (pos < 0) return false;
  const int lp = pos / c.page_size, slot = pos - lp * c.page_size;
  const int page = lp < c.max_pages ? c.page_table[static_cast<long long>(b) * c.max_pages + lp] : -1;
  if (page < 0 || page >= c.num_pages) {
    if (report && status != nullptr) atomicCAS(status, 0, kErrBadIndex);
    return false;
  }
  row = ((static_cast<long long>(page) * c.page_size + slot) * c.KV + h) * c.D;
  srow = ((static_cast<long long>(page) * c.KV + h) * c.page_size + slot) * (c.D / 32);
  return true;
}

// Index space: [token][K or V][head][D / 16], one thread each.
struct Unit {
  int tok, b, h, d0;
  bool is_v, first;
};
__device__ __forceinline__ Unit unit_of(unsigned idx, const MxCache& c, int T) {
  const unsigned per_head = c.D / 16, per_side = c.KV * per_head;
  const unsigned side = idx / per_side, rest = idx - side * per_side;
  Unit u;
  u.tok = side >> 1, u.is_v = side & 1;
  u.b = u.tok / T;
  u.h = rest / per_head;
  u.d0 = (rest - u.h * per_head) * 16;
  u.first = rest == 0;
  return u;
}

__global__ void __launch_bounds__(kThreads) kv_append_mx_kernel(const MxCache c, const int* __restrict__ positions, int T,
                                                                unsigned total, const KvRows kr, const KvRows vr,
                                                                int* status) {
  NC_PDL_PROLOGUE();
  const unsigned idx = blockIdx.x * kThreads + threadIdx.x;
  const bool live = idx < total;     // the shuffle below wants the whole warp
  const Unit u = unit_of(live ? idx : 0, c, T);
  const int pos = live ? positions[u.tok] : -1;
  uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (pos >= 0) {
    const KvRows& r = u.is_v ? vr : kr;
    const uint4* src = reinterpret_cast<const uint4*>(r.ptr + u.b * r.stride_b + (u.tok - u.b * T) * r.stride_t +
                                                      u.h * r.stride_h + u.d0);
    x[0] = src[0], x[1] = src[1];
  }
  const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
  uint32_t mx = 0;   // the larger magnitudes of even and odd channels, as 16-bit fields (magnitude bits order as numbers)
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = __vmaxu2(mx, w[i] & 0x7fff7fffu);
  mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  const uint32_t amax = max(mx & 0xffffu, mx >> 16);
  if (pos < 0) return;
  long long row, srow;
  if (!place(c, u.b, pos, u.h, status, u.first && !u.is_v, row, srow)) return;
  const uint32_t b = mx_scale_byte(amax);
  uint4 code = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);   // a block of NaN
  if (b != 255u) {
    const float inv = mx_inverse_scale(b);
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[2 * i] = bf16_lo(w[i]) * inv, f[2 * i + 1] = bf16_hi(w[i]) * inv;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = mx_to_e4m3x2(f[4 * i], f[4 * i + 1]) | (mx_to_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16);
    code = make_uint4(o[0], o[1], o[2], o[3]);
  }
  *reinterpret_cast<uint4*>((u.is_v ? c.v : c.k) + row + u.d0) = code;
  if ((u.d0 & 16) == 0) (u.is_v ? c.v_scale : c.k_scale)[srow + u.d0 / 32] = static_cast<uint8_t>(b);
}

__global__ void __launch_bounds__(kThreads) kv_read_mx_kernel(const MxCache c, const int* __restrict__ positions, int T,
                                                              unsigned total, __nv_bfloat16* __restrict__ k_out,
                                                              __nv_bfloat16* __restrict__ v_out, int* status) {
  NC_PDL_PROLOGUE();
  const unsigned idx = blockIdx.x * kThreads + threadIdx.x;
  if (idx >= total) return;
  const Unit u = unit_of(idx, c, T);
  uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  long long row, srow;
  if (place(c, u.b, positions[u.tok], u.h, status, u.first && !u.is_v, row, srow)) {
    const uint4 code = *reinterpret_cast<const uint4*>((u.is_v ? c.v : c.k) + row + u.d0);
    const uint32_t b = (u.is_v ? c.v_scale : c.k_scale)[srow + u.d0 / 32];
    const uint32_t f1 = mx_factor_first(b) * 0x10001u, f2 = mx_factor_second(b) * 0x10001u;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&code);
    uint32_t* r = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mx_spread(w[i], r[2 * i], r[2 * i + 1]);
      r[2 * i] = mul_bf16x2(mul_bf16x2(r[2 * i], f1), f2);
      r[2 * i + 1] = mul_bf16x2(mul_bf16x2(r[2 * i + 1], f1), f2);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>((u.is_v ? v_out : k_out) + (static_cast<long long>(u.tok) * c.KV + u.h) * c.D + u.d0);
  dst[0] = o[0], dst[1] = o[1];
}

const char* grid_of(const MxCache& c, int B, int T, unsigned& total, unsigned& blocks) {
  const long long n = 2LL * B * T * c.KV * (c.D / 16);
  if (n >= (1LL << 32) - kThreads) return "kv_mx: more than 2^32 units of 16 channels in one call";
  total = static_cast<unsigned>(n);
  blocks = (total + kThreads - 1) / kThreads;
  return nullptr;
}

}  // namespace

const char* kv_append_mx(const MxCache& c, const int* positions, int B, int T, const KvRows& k, const KvRows& v,
                         int* status, cudaStream_t s) {
  unsigned total, blocks;
  if (const char* e = grid_of(c, B, T, total, blocks)) return e;
  if (total == 0) return nullptr;
  const cudaError_t e = launch_maybe_pdl(kv_append_mx_kernel, dim3(blocks), dim3(kThreads), 0, s, c, positions, T, total, k,
                                         v, status);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* kv_read_mx(const MxCache& c, const int* positions, int B, int T, __nv_bfloat16* k_out, __nv_bfloat16* v_out,
                       int* status, cudaStream_t s) {
  unsigned total, blocks;
  if (const char* e = grid_of(c, B, T, total, blocks)) return e;
  if (total == 0) return nullptr;
  const cudaError_t e = launch_maybe_pdl(kv_read_mx_kernel, dim3(blocks), dim3(kThreads), 0, s, c, positions, T, total, k_out,
                                         v_out, status);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace nc
