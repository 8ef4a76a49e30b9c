// Host interface of the serving kernels: the MXFP8 key / value cache (kv_mx.cu), attention of new tokens over the
// paged cache (paged_rows.cu: few query rows per kv head, paged_chunk.cu: many), and sampling (sample.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nc {

// Code pools are E4M3 bytes [pages, page_size, KV, D], scale pools UE8M0 bytes [pages, KV, page_size, D / 32].
struct MxCache {
  uint8_t *k = nullptr, *v = nullptr;
  uint8_t *k_scale = nullptr, *v_scale = nullptr;
  const int* page_table = nullptr;  // [B, max_pages]
  int max_pages = 0, page_size = 16, num_pages = 0, KV = 0, D = 0;
};

// One row of K or V per (sequence, token): element (b, t, h, d) at ptr[b * stride_b + t * stride_t + h * stride_h + d].
struct KvRows {
  const __nv_bfloat16* ptr = nullptr;
  long long stride_b = 0, stride_t = 0, stride_h = 0;  // elements, multiples of 8
};

// Rows at absolute positions[B * T] (negative: skipped) are quantised into their pages. A position past the page table
// or a page outside the pool is not written and records code 7 in `status`.
const char* kv_append_mx(const MxCache& c, const int* positions, int B, int T, const KvRows& k, const KvRows& v,
                         int* status, cudaStream_t s);
// The inverse: dense bf16 [B, T, KV, D]; rows of a negative position are zero (and of an unusable one: with code 7).
const char* kv_read_mx(const MxCache& c, const int* positions, int B, int T, __nv_bfloat16* k_out, __nv_bfloat16* v_out,
                       int* status, cudaStream_t s);

struct PagedAttnArgs {
  int B = 0, T = 0, H = 0, KV = 0, D = 0;
  const __nv_bfloat16* q = nullptr;  // (b, t, h, d) at q[b * q_stride_b + t * q_stride_t + h * q_stride_h + d]
  long long q_stride_b = 0, q_stride_t = 0, q_stride_h = 0;
  const void *k_pool = nullptr, *v_pool = nullptr;              // bf16, or E4M3 codes when the scales are given
  const uint8_t *k_scale = nullptr, *v_scale = nullptr;
  const int* page_table = nullptr;                              // [B, max_pages]
  int max_pages = 0, page_size = 16, num_pages = 0;
  const int* seq_lens = nullptr;                                // [B], new tokens included
  const int* q_lens = nullptr;                                  // [B]; null: T for every sequence
  int window_left = -1;
  float scale = 1.0f;
  __nv_bfloat16* out = nullptr;                                 // dense [B, T, H, D]
  // Workspace for sequences whose keys are split over several CTAs (see the *_plan functions), or null for one split.
  float *part_o = nullptr, *part_ml = nullptr;
  int splits = 1, split_keys = 0;
  int* status = nullptr;
};

// Work split: keys per run and the floats of workspace it needs (0: none).
struct PagedPlan {
  int splits = 1, split_keys = 0;
  long long part_o = 0, part_ml = 0;
};
PagedPlan paged_rows_plan(const PagedAttnArgs& a);
const char* paged_rows_attention(const PagedAttnArgs& a, cudaStream_t s);
// Whether the rows make a grid that can be launched.
bool paged_rows_can(const PagedAttnArgs& a);
// The same for many rows per kv head: whether it can take these arguments, and whether it is the faster one for them.
bool paged_chunk_can(const PagedAttnArgs& a);
bool paged_chunk_takes(const PagedAttnArgs& a);
PagedPlan paged_chunk_plan(const PagedAttnArgs& a);
const char* paged_chunk_attention(const PagedAttnArgs& a, cudaStream_t s);

struct SampleArgs {
  const void* logits = nullptr;  // bf16 or fp32 rows, leading dimension ld
  bool bf16 = false;
  long long ld = 0;
  int rows = 0, vocab = 0;
  const float* u = nullptr;      // [rows]
  // one value per row, or null for the number beside it
  const float *temperature_rows = nullptr, *top_p_rows = nullptr, *min_p_rows = nullptr;
  const int* top_k_rows = nullptr;
  float temperature = 1.0f, top_p = 1.0f, min_p = 0.0f;
  int top_k = 0;
  long long* out = nullptr;      // [rows]
};
const char* sample_rows(const SampleArgs& a, cudaStream_t s);

}  // namespace nc
