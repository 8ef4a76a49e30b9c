// The MXFP8 key / value cache: rows are quantised as they are written into their pages, and read back as bf16.
//
// A block is 32 channels of one token and head: code = e4m3(x * 2^(127 - b)), value = code * 2^(b - 127) with b from the
// block's largest magnitude (mx_cache.cuh). Scales being powers of two, scaling is exact in both directions and the code
// is the only rounding. Both kernels only move bytes (append: 2 read, 1 + 1/32 written per element; read: the reverse),
// but at a few hundred bytes a row they run out of instructions before bandwidth if every thread works out its own place:
// a warp takes a token (several, where they are narrow), finds the place once, and its lanes go over the key AND value
// row in pieces of 8 channels, neighbouring lanes on neighbouring pieces. Four lanes share a block and exchange their
// maxima by two shuffles. The scale pool is laid out [page, head, token, block]: the scales of one page and head, which
// the attention kernels read together, are contiguous. Measured (B200): append and read of 16 prompts up to 2048, 10 heads
// of 128, 83 us for both, 4.4 TB/s; a thread that found its own place took 104.
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
constexpr int kBatch = 4;   // pieces of a row that a lane has in flight

// The lanes of a warp: `per` of them to a token, 8 channels each at a time, and so many tokens per warp.
struct Split {
  int units, per, tokens;
};

struct Place {
  long long row, srow;   // of the code pools (the token's row) and scale pools (its first head); row < 0: no usable place
  int tok, b, t, pos;    // pos < 0: skipped, or not a token of the call
  int first;             // the lane's first piece
  bool live;
};
__device__ __forceinline__ Place find(const MxCache& c, const int* positions, int B, int T, const Split& s) {
  Place p;
  const int lane = threadIdx.x & 31, warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int sub = s.tokens > 1 ? lane / s.per : 0;
  p.first = lane - sub * s.per;
  p.tok = warp * s.tokens + sub;
  p.live = sub < s.tokens && p.tok < B * T;
  p.pos = p.live ? positions[p.tok] : -1;
  p.b = T == 1 ? p.tok : p.tok / T;
  p.t = p.tok - p.b * T;
  return p;
}
__device__ __forceinline__ void look_up(const MxCache& c, int* status, Place& p) {
  p.row = p.srow = -1;
  if (p.pos < 0) return;
  const int lp = p.pos / c.page_size, slot = p.pos - lp * c.page_size;
  const int page = lp < c.max_pages ? c.page_table[static_cast<long long>(p.b) * c.max_pages + lp] : -1;
  if (page < 0 || page >= c.num_pages) {
    if (p.first == 0 && status != nullptr) atomicCAS(status, 0, kErrBadIndex);
    return;
  }
  p.row = (static_cast<long long>(page) * c.page_size + slot) * c.KV * c.D;
  p.srow = (static_cast<long long>(page) * c.KV * c.page_size + slot) * (c.D / 32);
}

// Eight values of a block of four neighbouring lanes -> eight codes and the block's scale byte.
__device__ __forceinline__ uint2 encode(const uint4& x, uint32_t& b) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t mx = 0;   // the larger magnitudes of even and odd channels, as 16-bit fields (magnitude bits order as numbers)
#pragma unroll
  for (int i = 0; i < 4; ++i) mx = __vmaxu2(mx, w[i] & 0x7fff7fffu);
  mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  b = mx_scale_byte(max(mx & 0xffffu, mx >> 16));
  if (b == 255u) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);   // a block of NaN
  const float inv = mx_inverse_scale(b);
  const float f[8] = {bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1]), bf16_lo(w[2]), bf16_hi(w[2]), bf16_lo(w[3]), bf16_hi(w[3])};
  return mx_pack8(f, inv);
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv_append_mx_kernel(const MxCache c, const int* __restrict__ positions, int B, int T,
                                                                const Split s, const KvRows kr, const KvRows vr, int* status) {
  NC_PDL_PROLOGUE();
  Place p = find(c, positions, B, T, s);
  const __nv_bfloat16* ks = kr.ptr + p.b * kr.stride_b + p.t * kr.stride_t;
  const __nv_bfloat16* vs = vr.ptr + p.b * vr.stride_b + p.t * vr.stride_t;
  bool looked = false;
  // every lane of the warp goes round as often: the shuffles want all of them
  for (int u0 = 0; u0 < s.units; u0 += kBatch * s.per) {
    uint4 xk[kBatch], xv[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = u0 + i * s.per + p.first, h = u / (D / 8), d0 = u % (D / 8) * 8;
      xk[i] = xv[i] = make_uint4(0, 0, 0, 0);
      if (u < s.units && p.pos >= 0) {
        xk[i] = __ldcs(reinterpret_cast<const uint4*>(ks + h * kr.stride_h + d0));
        xv[i] = __ldcs(reinterpret_cast<const uint4*>(vs + h * vr.stride_h + d0));
      }
    }
    if (!looked) look_up(c, status, p), looked = true;   // (the first rows are on their way meanwhile)
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = u0 + i * s.per + p.first, h = u / (D / 8), d0 = u % (D / 8) * 8;
      if (u0 + i * s.per >= s.units) break;              // the same for every lane
      uint32_t bk, bv;
      const uint2 ck = encode(xk[i], bk), cv = encode(xv[i], bv);
      if (u < s.units && p.row >= 0) {
        *reinterpret_cast<uint2*>(c.k + p.row + u * 8) = ck;
        *reinterpret_cast<uint2*>(c.v + p.row + u * 8) = cv;
        if ((d0 & 31) == 0) {
          const long long at = p.srow + static_cast<long long>(h) * c.page_size * (D / 32) + d0 / 32;
          c.k_scale[at] = static_cast<uint8_t>(bk), c.v_scale[at] = static_cast<uint8_t>(bv);
        }
      }
    }
  }
}

__device__ __forceinline__ uint4 decode(const uint2& code, uint32_t b) {
  const uint32_t f1 = mx_factor_first(b) * 0x10001u, f2 = mx_factor_second(b) * 0x10001u;
  uint32_t r[4];
  mx_spread(code.x, r[0], r[1]);
  mx_spread(code.y, r[2], r[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = mul_bf16x2(mul_bf16x2(r[i], f1), f2);
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv_read_mx_kernel(const MxCache c, const int* __restrict__ positions, int B, int T,
                                                              const Split s, __nv_bfloat16* __restrict__ k_out,
                                                              __nv_bfloat16* __restrict__ v_out, int* status) {
  NC_PDL_PROLOGUE();
  Place p = find(c, positions, B, T, s);
  if (!p.live) return;
  look_up(c, status, p);
  const long long out = static_cast<long long>(p.tok) * c.KV * D;
  for (int u0 = p.first; u0 < s.units; u0 += kBatch * s.per) {
    uint2 ck[kBatch], cv[kBatch];
    uint32_t bk[kBatch], bv[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = u0 + i * s.per, h = u / (D / 8), d0 = u % (D / 8) * 8;
      ck[i] = cv[i] = make_uint2(0, 0), bk[i] = bv[i] = 127;
      if (u < s.units && p.row >= 0) {
        ck[i] = *reinterpret_cast<const uint2*>(c.k + p.row + u * 8), cv[i] = *reinterpret_cast<const uint2*>(c.v + p.row + u * 8);
        const long long at = p.srow + static_cast<long long>(h) * c.page_size * (D / 32) + d0 / 32;
        bk[i] = c.k_scale[at], bv[i] = c.v_scale[at];
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = u0 + i * s.per;
      if (u >= s.units) break;
      __stcs(reinterpret_cast<uint4*>(k_out + out + u * 8), decode(ck[i], bk[i]));
      __stcs(reinterpret_cast<uint4*>(v_out + out + u * 8), decode(cv[i], bv[i]));
    }
  }
}

Split split_of(const MxCache& c) {
  Split s;
  s.units = c.KV * (c.D / 8);
  s.per = s.units < 32 ? s.units : 32;   // a multiple of 8: blocks of four lanes stay together
  s.tokens = 32 / s.per;
  return s;
}
unsigned blocks_of(const Split& s, int B, int T) {
  const long long per_cta = static_cast<long long>(s.tokens) * (kThreads / 32);
  return static_cast<unsigned>((static_cast<long long>(B) * T + per_cta - 1) / per_cta);
}

}  // namespace

const char* kv_append_mx(const MxCache& c, const int* positions, int B, int T, const KvRows& k, const KvRows& v,
                         int* status, cudaStream_t s) {
  if (B == 0 || T == 0) return nullptr;
  const Split h = split_of(c);
  const cudaError_t e = launch_maybe_pdl(c.D == 128 ? kv_append_mx_kernel<128> : kv_append_mx_kernel<64>,
                                         dim3(blocks_of(h, B, T)), dim3(kThreads), 0, s, c, positions, B, T, h, k, v, status);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* kv_read_mx(const MxCache& c, const int* positions, int B, int T, __nv_bfloat16* k_out, __nv_bfloat16* v_out,
                       int* status, cudaStream_t s) {
  if (B == 0 || T == 0) return nullptr;
  const Split h = split_of(c);
  const cudaError_t e = launch_maybe_pdl(c.D == 128 ? kv_read_mx_kernel<128> : kv_read_mx_kernel<64>, dim3(blocks_of(h, B, T)),
                                         dim3(kThreads), 0, s, c, positions, B, T, h, k_out, v_out, status);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace nc
