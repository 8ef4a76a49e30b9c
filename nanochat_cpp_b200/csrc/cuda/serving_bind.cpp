// Tensor-level wrappers of the serving kernels: MXFP8 cache, attention over pages, sampling.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "serving.h"

namespace ncbind {
int* device_status(int device);   // bindings.cpp: the device's status word
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

inline bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
inline void same_device(const Tensor& t, const Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device(), op, ": ", name, " must be on the device of the pools");
}

void check_pools(const char* op, const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs) {
  const bool mx = ks.has_value();
  TORCH_CHECK(vs.has_value() == mx, op, ": give both scales or neither");
  const auto type = mx ? torch::kUInt8 : torch::kBFloat16;
  for (const Tensor* t : {&k, &v}) {
    TORCH_CHECK(t->is_cuda() && t->dim() == 4 && t->is_contiguous() && t->scalar_type() == type && aligned16(*t), op,
                ": pools must be contiguous ", mx ? "uint8" : "bf16", " [pages, page_size, KV, D], 16-byte aligned");
  }
  TORCH_CHECK(v.sizes() == k.sizes(), op, ": v_pool must have the shape of k_pool");
  same_device(v, k, op, "v_pool");
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, op, ": head_dim must be 64 or 128");
  TORCH_CHECK(k.size(0) > 0 && k.size(0) < (1LL << 31) && k.size(1) > 0 && k.size(1) < (1 << 20) && k.size(2) > 0, op, ": pool sizes out of range");
  if (!mx) return;
  for (const OptTensor* s : {&ks, &vs}) {
    TORCH_CHECK((*s)->scalar_type() == torch::kUInt8 && (*s)->dim() == 4 && (*s)->is_contiguous() && aligned16(**s) &&
                    (*s)->size(0) == k.size(0) && (*s)->size(1) == k.size(2) && (*s)->size(2) == k.size(1) &&
                    (*s)->size(3) == k.size(3) / 32,
                op, ": scales must be contiguous uint8 [pages, KV, page_size, D / 32], 16-byte aligned");
    same_device(**s, k, op, "scale");
  }
}

void check_table(const char* op, const Tensor& table, int64_t B, const Tensor& like) {
  same_device(table, like, op, "page_table");
  TORCH_CHECK(table.scalar_type() == torch::kInt32 && table.dim() == 2 && table.is_contiguous() && table.size(0) == B &&
                  table.size(1) > 0 && table.size(1) < (1LL << 31),
              op, ": page_table must be contiguous int32 [B, max_pages]");
}

nc::MxCache mx_cache(const char* op, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                     const Tensor& table, const Tensor& positions) {
  check_pools(op, k, v, ks, vs);
  same_device(positions, k, op, "positions");
  TORCH_CHECK(positions.scalar_type() == torch::kInt32 && positions.dim() == 2 && positions.is_contiguous() &&
                  positions.numel() < (1LL << 30),
              op, ": positions must be contiguous int32 [B, T]");
  check_table(op, table, positions.size(0), k);
  nc::MxCache c;
  c.k = k.data_ptr<uint8_t>(), c.v = v.data_ptr<uint8_t>();
  c.k_scale = ks.data_ptr<uint8_t>(), c.v_scale = vs.data_ptr<uint8_t>();
  c.page_table = table.data_ptr<int>();
  c.max_pages = table.size(1), c.page_size = k.size(1), c.num_pages = k.size(0), c.KV = k.size(2), c.D = k.size(3);
  return c;
}

// [B, T, heads, D] rows that allow 16-byte loads and tensor maps; a view that does not is copied (by clone: contiguous()
// returns a dense view as it is, whatever its address).
Tensor row_view(const char* op, const char* name, const Tensor& t, int dim = 4) {
  TORCH_CHECK(t.dim() == dim && t.scalar_type() == torch::kBFloat16, op, ": ", name, " must be bf16 ",
              dim == 4 ? "[B, T, heads, D]" : "[B, heads, D]");
  bool ok = t.stride(dim - 1) == 1 && aligned16(t);
  for (int i = 0; i < dim - 1; ++i) ok = ok && t.stride(i) > 0 && t.stride(i) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

nc::KvRows kv_rows(const Tensor& t) {
  nc::KvRows r;
  r.ptr = reinterpret_cast<const __nv_bfloat16*>(t.data_ptr());
  r.stride_b = t.stride(0), r.stride_t = t.stride(1), r.stride_h = t.stride(2);
  return r;
}

void kv_append_mx(Tensor& k_pool, Tensor& v_pool, Tensor& k_scale, Tensor& v_scale, const Tensor& page_table,
                  const Tensor& positions, const Tensor& k_new, const Tensor& v_new) {
  const char* op = "kv_append_mx";
  const c10::cuda::CUDAGuard g(k_pool.device());
  const nc::MxCache c = mx_cache(op, k_pool, v_pool, k_scale, v_scale, page_table, positions);
  const int B = positions.size(0), T = positions.size(1);
  for (const Tensor* t : {&k_new, &v_new}) {
    same_device(*t, k_pool, op, "new rows");
    TORCH_CHECK(t->dim() == 4 && t->size(0) == B && t->size(1) == T && t->size(2) == c.KV && t->size(3) == c.D, op,
                ": new rows must be [B, T, KV, D]");
  }
  const Tensor k = row_view(op, "k_new", k_new), v = row_view(op, "v_new", v_new);
  const char* err = nc::kv_append_mx(c, positions.data_ptr<int>(), B, T, kv_rows(k), kv_rows(v),
                                     ncbind::device_status(k_pool.get_device()), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(err == nullptr, err);
}

std::vector<Tensor> kv_read_mx(const Tensor& k_pool, const Tensor& v_pool, const Tensor& k_scale, const Tensor& v_scale,
                               const Tensor& page_table, const Tensor& positions) {
  const c10::cuda::CUDAGuard g(k_pool.device());
  const nc::MxCache c = mx_cache("kv_read_mx", k_pool, v_pool, k_scale, v_scale, page_table, positions);
  const int B = positions.size(0), T = positions.size(1);
  const auto opt = k_pool.options().dtype(torch::kBFloat16);
  Tensor k = at::empty({B, T, c.KV, c.D}, opt), v = at::empty({B, T, c.KV, c.D}, opt);
  const char* err = nc::kv_read_mx(c, positions.data_ptr<int>(), B, T, reinterpret_cast<__nv_bfloat16*>(k.data_ptr()),
                                   reinterpret_cast<__nv_bfloat16*>(v.data_ptr()),
                                   ncbind::device_status(k_pool.get_device()), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(err == nullptr, err);
  return {k, v};
}

// q [B, T, H, D], or [B, H, D] for one token each (any strides that are multiples of 8); the result is dense and of q's
// shape.
Tensor paged_attention(const char* op, const Tensor& q_in, const Tensor& k_pool, const Tensor& v_pool, const Tensor& page_table,
                       const Tensor& seq_lens, const OptTensor& q_lens, int64_t window_left, double scale,
                       const OptTensor& k_scale, const OptTensor& v_scale, int64_t variant) {
  const c10::cuda::CUDAGuard g(k_pool.device());
  check_pools(op, k_pool, v_pool, k_scale, v_scale);
  same_device(q_in, k_pool, op, "q");
  const bool one = q_in.dim() == 3;
  nc::PagedAttnArgs a;
  const int h = one ? 1 : 2;   // dimension of the heads
  // row numbers are ints in the kernels: T * H with room for the last tile
  TORCH_CHECK(q_in.dim() == h + 2 && q_in.size(0) <= 65535 && q_in.size(h) < (1 << 16) &&
                  (one || (q_in.size(1) < (1 << 24) && q_in.size(1) * q_in.size(h) < (1LL << 30))) &&
                  q_in.numel() / std::max<int64_t>(q_in.size(h + 1), 1) < (1LL << 32),
              op, ": q is too large");
  a.B = q_in.size(0), a.T = one ? 1 : q_in.size(1), a.H = q_in.size(h), a.D = q_in.size(h + 1), a.KV = k_pool.size(2);
  TORCH_CHECK(k_pool.size(3) == a.D && a.H > 0 && a.H % a.KV == 0, op,
              ": heads must be a multiple of kv heads, and q and the pools must have one head_dim");
  check_table(op, page_table, a.B, k_pool);
  auto check_lens = [&](const Tensor& t, const char* name) {
    same_device(t, k_pool, op, name);
    TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.size(0) == a.B && t.is_contiguous(), op, ": ", name,
                " must be contiguous int32 [B]");
  };
  check_lens(seq_lens, "seq_lens");
  if (q_lens.has_value()) check_lens(*q_lens, "q_lens");
  a.page_size = k_pool.size(1), a.num_pages = k_pool.size(0), a.scale = static_cast<float>(scale);
  a.max_pages = page_table.size(1);
  a.window_left = window_left < 0 ? -1 : static_cast<int>(std::min<int64_t>(window_left, 1 << 30));
  const bool can = nc::paged_chunk_can(a);
  TORCH_CHECK(variant >= 0 && variant <= 2 && (variant != 2 || can), op,
              ": variant must be 0 (by size), 1 (few rows) or 2 (many rows: page_size a multiple of 16, scale > 0)");
  const bool rows_can = nc::paged_rows_can(a);
  const bool chunk = variant == 0 ? nc::paged_chunk_takes(a) || (can && !rows_can) : variant == 2;
  TORCH_CHECK(chunk || rows_can, op, ": so many new tokens need pages of a multiple of 16 tokens and a scale above 0");
  const Tensor q = row_view(op, "q", q_in, one ? 3 : 4);
  Tensor out = at::empty(q.sizes(), q.options());
  if (out.numel() == 0) return out;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride_b = q.stride(0), a.q_stride_t = one ? a.H * static_cast<long long>(a.D) : q.stride(1), a.q_stride_h = q.stride(h);
  a.k_pool = k_pool.data_ptr(), a.v_pool = v_pool.data_ptr();
  if (k_scale.has_value()) a.k_scale = k_scale->data_ptr<uint8_t>(), a.v_scale = v_scale->data_ptr<uint8_t>();
  a.page_table = page_table.data_ptr<int>();
  a.seq_lens = seq_lens.data_ptr<int>();
  if (q_lens.has_value()) a.q_lens = q_lens->data_ptr<int>();
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.status = ncbind::device_status(k_pool.get_device());
  const nc::PagedPlan p = chunk ? nc::paged_chunk_plan(a) : nc::paged_rows_plan(a);
  a.splits = p.splits, a.split_keys = p.split_keys;
  Tensor work;
  if (p.splits > 1) {   // a buffer of its own per call: calls on other streams or in other graphs never share it
    work = at::empty({p.part_o + p.part_ml}, q.options().dtype(torch::kFloat32));
    a.part_o = work.data_ptr<float>(), a.part_ml = a.part_o + p.part_o;
  }
  const auto stream = at::cuda::getCurrentCUDAStream();
  const char* err = chunk ? nc::paged_chunk_attention(a, stream) : nc::paged_rows_attention(a, stream);
  TORCH_CHECK(err == nullptr, err);
  return out;
}

Tensor paged_chunk_attention(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& page_table,
                             const Tensor& seq_lens, const OptTensor& q_lens, int64_t window_left, double scale,
                             const OptTensor& k_scale, const OptTensor& v_scale, int64_t variant) {
  TORCH_CHECK(q.dim() == 4, "paged_chunk_attention: q must be [B, T, H, D]");
  return paged_attention("paged_chunk_attention", q, k_pool, v_pool, page_table, seq_lens, q_lens, window_left, scale,
                         k_scale, v_scale, variant);
}

Tensor paged_decode_attention_mx(const Tensor& q, const Tensor& k_pool, const Tensor& v_pool, const Tensor& k_scale,
                                 const Tensor& v_scale, const Tensor& page_table, const Tensor& seq_lens,
                                 int64_t window_left, double scale) {
  TORCH_CHECK(q.dim() == 3, "paged_decode_attention_mx: q must be [B, H, D]");
  return paged_attention("paged_decode_attention_mx", q, k_pool, v_pool, page_table, seq_lens, OptTensor(), window_left,
                         scale, k_scale, v_scale, 0);
}

Tensor sample_rows(const Tensor& logits, const Tensor& u, double temperature, int64_t top_k, double top_p, double min_p,
                   const OptTensor& temperature_rows, const OptTensor& top_k_rows, const OptTensor& top_p_rows,
                   const OptTensor& min_p_rows) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) > 0 && logits.stride(1) == 1 &&
                  (logits.scalar_type() == torch::kBFloat16 || logits.scalar_type() == torch::kFloat32) &&
                  logits.size(1) < (1 << 30) && logits.size(0) < (1LL << 31),
              "sample_rows: logits must be bf16 or fp32 [rows, vocab] with dense rows");
  const c10::cuda::CUDAGuard g(logits.device());
  const int64_t R = logits.size(0);
  auto rows = [&](const Tensor& t, torch::ScalarType type, const char* name) {
    same_device(t, logits, "sample_rows", name);
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.size(0) == R && t.is_contiguous(), "sample_rows: ", name,
                " must be a number or a contiguous ", type == torch::kInt32 ? "int32" : "fp32", " [rows] tensor");
  };
  rows(u, torch::kFloat32, "u");
  nc::SampleArgs a;
  a.logits = logits.data_ptr();
  a.bf16 = logits.scalar_type() == torch::kBFloat16;
  a.ld = logits.stride(0);
  a.rows = R, a.vocab = logits.size(1);
  a.u = u.data_ptr<float>();
  a.temperature = temperature, a.top_p = top_p, a.min_p = min_p;
  a.top_k = static_cast<int>(std::max<int64_t>(std::min<int64_t>(top_k, 1 << 30), 0));
  if (temperature_rows.has_value()) rows(*temperature_rows, torch::kFloat32, "temperature"), a.temperature_rows = temperature_rows->data_ptr<float>();
  if (top_p_rows.has_value()) rows(*top_p_rows, torch::kFloat32, "top_p"), a.top_p_rows = top_p_rows->data_ptr<float>();
  if (min_p_rows.has_value()) rows(*min_p_rows, torch::kFloat32, "min_p"), a.min_p_rows = min_p_rows->data_ptr<float>();
  if (top_k_rows.has_value()) rows(*top_k_rows, torch::kInt32, "top_k"), a.top_k_rows = top_k_rows->data_ptr<int>();
  Tensor out = at::empty({R}, logits.options().dtype(torch::kInt64));
  a.out = reinterpret_cast<long long*>(out.data_ptr<int64_t>());
  const char* err = nc::sample_rows(a, at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(err == nullptr, err);
  return out;
}

}  // namespace

void register_serving(pybind11::module_& m) {
  m.def("kv_append_mx", &kv_append_mx);
  m.def("kv_read_mx", &kv_read_mx);
  m.def("paged_chunk_attention", &paged_chunk_attention);
  m.def("paged_decode_attention_mx", &paged_decode_attention_mx);
  m.def("sample_rows", &sample_rows);
}
