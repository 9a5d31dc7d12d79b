// Python bindings of the paged 8-bit cache kernels and the batched sampler (part of `_C`).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "kernels/paged8.h"
#include "kernels/sample.h"

namespace {

#define HCP_CHECK_OK(err) TORCH_CHECK((err) == nullptr, "hcp kernel: ", (err))

using c10::optional;
using torch::Tensor;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_array(const Tensor& t, const char* name, torch::ScalarType type, int64_t dim, const torch::Device& dev) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
  // (numbers in messages as text: streaming them into the check's message crashed with this torch build)
  TORCH_CHECK(t.dim() == dim && t.is_contiguous(), name, " must be a contiguous ", std::to_string(dim), "-d tensor");
}

int dtype_of(const Tensor& t, const char* name, bool f32) {
  if (t.scalar_type() == torch::kBFloat16) return hcp::kv8::kBF16;
  if (t.scalar_type() == torch::kHalf) return hcp::kv8::kF16;
  TORCH_CHECK(f32 && t.scalar_type() == torch::kFloat32, name, " must be bfloat16", f32 ? ", float16 or float32" : " or float16");
  return hcp::kv8::kF32;
}

int* status_ptr(const optional<Tensor>& t, const torch::Device& dev) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->device() == dev && t->scalar_type() == torch::kInt32 && t->is_contiguous() && t->numel() >= 4,
              "status must be a contiguous int32 tensor of 4 or more elements on ", dev);
  return t->data_ptr<int>();
}

hcp::kv8::Cache cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  TORCH_CHECK(k.is_cuda() && v.device() == k.device() && ks.device() == k.device() && vs.device() == k.device(),
              "the cache's tensors must be on one CUDA device");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.scalar_type() == v.scalar_type(),
              "k and v must be [pages, kv_heads, page, head_dim] of one type, shape and strides");
  TORCH_CHECK(k.scalar_type() == torch::kFloat8_e4m3fn || k.scalar_type() == torch::kInt8, "the cache holds float8_e4m3fn or int8");
  // (before anything divides by the head count)
  TORCH_CHECK(k.numel() > 0, "the cache must have a page, a KV head, tokens and dims");
  TORCH_CHECK(k.stride(3) == 1, "cache rows must be contiguous");
  TORCH_CHECK(ks.dim() == 2 && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && ks.sizes() == vs.sizes() &&
                  ks.strides() == vs.strides() && ks.scalar_type() == torch::kFloat32 && vs.scalar_type() == torch::kFloat32,
              "the scales must be float32 [pages, kv_heads], k's and v's alike");
  hcp::kv8::Cache c{};
  c.k = static_cast<uint8_t*>(k.data_ptr());
  c.v = static_cast<uint8_t*>(v.data_ptr());
  c.k_scale = ks.data_ptr<float>();
  c.v_scale = vs.data_ptr<float>();
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.token_stride = k.stride(2);
  c.scale_page_stride = ks.stride(0);
  c.scale_head_stride = ks.stride(1);
  TORCH_CHECK(k.size(0) < (1ll << 31) && k.size(1) < (1 << 16), "too many pages or KV heads");
  c.pages = int(k.size(0));
  c.Hkv = int(k.size(1));
  c.P = int(k.size(2));
  c.D = int(k.size(3));
  c.code = k.scalar_type() == torch::kInt8 ? hcp::kv8::kInt8 : hcp::kv8::kE4M3;
  return c;
}

int sm_count(int dev) { return at::cuda::getDeviceProperties(dev)->multiProcessorCount; }

void plan_step(const Tensor& add, const Tensor& kv_len, const Tensor& table, const Tensor& ring, const Tensor& counters, int64_t page,
               const Tensor& cu, const Tensor& row, const Tensor& pos, const Tensor& slot, const Tensor& unit,
               const Tensor& kv_len_out, const Tensor& counters_out, const Tensor& info) {
  const auto dev = add.device();
  TORCH_CHECK(add.is_cuda(), "add must be a CUDA tensor");
  check_array(add, "add", torch::kInt32, 1, dev);
  check_array(kv_len, "kv_len", torch::kInt32, 1, dev);
  check_array(table, "block_table", torch::kInt32, 2, dev);
  check_array(ring, "ring", torch::kInt32, 1, dev);
  check_array(counters, "counters", torch::kInt64, 1, dev);
  check_array(cu, "cu", torch::kInt32, 1, dev);
  check_array(row, "row", torch::kInt32, 1, dev);
  check_array(pos, "pos", torch::kInt32, 1, dev);
  check_array(slot, "slot", torch::kInt64, 1, dev);
  check_array(unit, "unit", torch::kInt32, 2, dev);
  check_array(kv_len_out, "kv_len (out)", torch::kInt32, 1, dev);
  check_array(counters_out, "counters (out)", torch::kInt64, 1, dev);
  check_array(info, "info", torch::kInt32, 1, dev);
  const int64_t R = add.size(0), T = row.size(0);
  TORCH_CHECK(kv_len.size(0) == R && table.size(0) == R && kv_len_out.size(0) == R && cu.size(0) == R + 1,
              "add, kv_len, block_table and cu must have one entry per row");
  TORCH_CHECK(pos.size(0) == T && slot.size(0) == T, "row, pos and slot must have one entry per token");
  TORCH_CHECK(unit.size(1) == 4, "unit must be [units, 4]");
  TORCH_CHECK(counters.size(0) == 2 && counters_out.size(0) == 2 && info.size(0) == 4, "counters must have 2 entries, info 4");
  TORCH_CHECK(page >= 1 && page <= (1 << 20), "page must be 1 to 2^20 tokens");
  TORCH_CHECK(R <= hcp::kv8::kPlanMaxRows && T < (1ll << 30) && unit.size(0) < (1ll << 30) && table.size(1) < (1ll << 31) && ring.size(0) < (1ll << 31),
              "plan_step: at most ", std::to_string(hcp::kv8::kPlanMaxRows), " rows, fewer than 2^30 tokens and units, and every other size below 2^31");
  TORCH_CHECK(unit.size(0) >= std::min(T, T / page + 2 * R), "unit must have min(tokens, tokens / page + 2 rows) entries");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(row.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(pos.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(slot.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(unit.data_ptr()) % 16 == 0,
              "row, pos, slot and unit must start on 16-byte boundaries");
  const c10::cuda::CUDAGuard g(dev);
  hcp::kv8::PlanArgs a{};
  a.add = add.data_ptr<int>();
  a.kv_len = kv_len.data_ptr<int>();
  a.table = table.data_ptr<int>();
  a.ring = ring.data_ptr<int>();
  a.counters = reinterpret_cast<const long long*>(counters.data_ptr<int64_t>());
  a.R = int(R);
  a.width = int(table.size(1));
  a.P = int(page);
  a.ring_size = int(ring.size(0));
  a.max_tokens = int(T);
  a.max_units = int(unit.size(0));
  a.cu = cu.data_ptr<int>();
  a.row = row.data_ptr<int>();
  a.pos = pos.data_ptr<int>();
  a.slot = reinterpret_cast<long long*>(slot.data_ptr<int64_t>());
  a.unit = reinterpret_cast<int4*>(unit.data_ptr<int>());
  a.kv_len_out = kv_len_out.data_ptr<int>();
  a.counters_out = reinterpret_cast<long long*>(counters_out.data_ptr<int64_t>());
  a.info = info.data_ptr<int>();
  HCP_CHECK_OK(hcp::kv8::plan_step(a, cur_stream()));
}

std::tuple<Tensor, int> rope_append_kv8(const Tensor& x, const Tensor& cos_t, const Tensor& sin_t, const Tensor& pos, const Tensor& unit,
                       const Tensor& table, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t heads,
                       optional<Tensor> q_out, optional<Tensor> status) {
  hcp::kv8::AppendArgs a{};
  a.c = cache_of(k, v, ks, vs);
  const auto dev = k.device();
  const int64_t D = a.c.D, T = x.size(0);
  TORCH_CHECK(x.device() == dev && x.dim() == 2 && x.stride(1) == 1, "qkv must be [tokens, (heads + 2 kv_heads) * head_dim] with contiguous rows");
  TORCH_CHECK(heads >= 1 && heads < (1 << 16) && x.size(1) == (heads + 2 * a.c.Hkv) * D, "qkv must have heads + 2 kv_heads heads a row");
  check_array(cos_t, "cos", torch::kFloat32, 2, dev);
  check_array(sin_t, "sin", torch::kFloat32, 2, dev);
  TORCH_CHECK(cos_t.size(1) == D / 2 && cos_t.sizes() == sin_t.sizes() && cos_t.size(0) >= 1, "cos and sin must be [positions, head_dim / 2]");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(cos_t.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(sin_t.data_ptr()) % 16 == 0,
              "cos and sin must start on 16-byte boundaries");
  check_array(pos, "pos", torch::kInt32, 1, dev);
  check_array(unit, "unit", torch::kInt32, 2, dev);
  check_array(table, "block_table", torch::kInt32, 2, dev);
  TORCH_CHECK(pos.size(0) >= T, "pos must have one entry per token");
  TORCH_CHECK(unit.size(1) == 4 && reinterpret_cast<uintptr_t>(unit.data_ptr()) % 16 == 0, "unit must be [units, 4], 16-byte aligned");
  TORCH_CHECK(T < (1ll << 31) && unit.size(0) < (1ll << 31) && cos_t.size(0) < (1ll << 31), "rope_append_kv8: too many tokens");
  const c10::cuda::CUDAGuard g(dev);
  a.dtype = dtype_of(x, "qkv", true);
  Tensor out;
  if (q_out.has_value() && q_out->defined()) {
    out = *q_out;
    TORCH_CHECK(out.device() == dev && out.is_contiguous() && out.numel() == T * heads * D, "q_out must be contiguous [tokens, heads, head_dim]");
  } else {
    out = torch::empty({T, heads, D}, x.options().dtype(a.dtype == hcp::kv8::kF32 ? torch::kBFloat16 : x.scalar_type()));
  }
  a.q_dtype = dtype_of(out, "q_out", false);
  a.x = x.data_ptr();
  a.row_stride = x.stride(0);
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.max_pos = int(cos_t.size(0));
  a.pos = pos.data_ptr<int>();
  a.unit = reinterpret_cast<const int4*>(unit.data_ptr<int>());
  a.table = table.data_ptr<int>();
  a.T = int(T);
  a.H = int(heads);
  a.U = int(unit.size(0));
  a.R = int(table.size(0));
  a.width = int(table.size(1));
  a.q_out = out.data_ptr();
  a.status = status_ptr(status, dev);
  a.num_sms = sm_count(dev.index());
  int launched = 0;
  HCP_CHECK_OK(hcp::kv8::rope_append(a, cur_stream(), &launched));
  return {out, launched};
}

std::tuple<Tensor, Tensor> gather_kv8(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& table, int64_t n,
                                      const optional<Tensor>& k_buf, const optional<Tensor>& v_buf) {
  hcp::kv8::GatherArgs a{};
  a.c = cache_of(k, v, ks, vs);
  const auto dev = k.device();
  check_array(table, "block_table row", torch::kInt32, 1, dev);
  // (the kernel numbers a head's 16-byte pieces in 32 bits; before any buffer is made)
  TORCH_CHECK(n >= 0 && n * a.c.D < (1ll << 35) - (1ll << 12), "gather_kv8: rows to gather out of range");
  const c10::cuda::CUDAGuard g(dev);
  TORCH_CHECK(k_buf.has_value() == v_buf.has_value(), "give both output buffers or none");
  Tensor k_out, v_out;
  if (k_buf.has_value()) {
    k_out = *k_buf;
    v_out = *v_buf;
  } else {
    const auto opt = k.options().dtype(torch::kBFloat16);
    k_out = torch::empty({a.c.Hkv, n, a.c.D}, opt);
    v_out = torch::empty({a.c.Hkv, n, a.c.D}, opt);
  }
  for (const Tensor* o : {&k_out, &v_out}) {
    TORCH_CHECK(o->device() == dev && o->scalar_type() == torch::kBFloat16 && o->dim() == 3 && o->size(0) == a.c.Hkv && o->size(1) >= n &&
                    o->size(2) == a.c.D && o->stride(2) == 1 && o->stride(1) == a.c.D && o->stride(0) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(o->data_ptr()) % 16 == 0,
                "the outputs must be bfloat16 [kv_heads, rows or more, head_dim] with contiguous rows");
  }
  TORCH_CHECK(k_out.strides() == v_out.strides(), "the outputs must have the same strides");
  a.table = table.data_ptr<int>();
  a.width = int(table.size(0));
  a.n = int(n);
  a.k_out = k_out.data_ptr();
  a.v_out = v_out.data_ptr();
  a.out_head_stride = k_out.stride(0);
  HCP_CHECK_OK(hcp::kv8::gather(a, cur_stream()));
  return {k_out, v_out};
}

std::tuple<Tensor, Tensor> attention_kv8(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                                         const Tensor& table, const Tensor& kv_len, optional<Tensor> cu, int64_t max_q, double scale,
                                         optional<Tensor> out, bool want_lse, optional<Tensor> status) {
  hcp::kv8::AttnArgs a{};
  a.c = cache_of(k, v, ks, vs);
  const auto dev = k.device();
  TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.size(2) == a.c.D && q.stride(2) == 1, "q must be [tokens, heads, head_dim] with contiguous heads");
  check_array(table, "block_table", torch::kInt32, 2, dev);
  check_array(kv_len, "kv_len", torch::kInt32, 1, dev);
  const int64_t T = q.size(0), H = q.size(1), B = kv_len.size(0);
  TORCH_CHECK(table.size(0) == B && table.size(1) >= 1, "block_table must have one row per request");
  TORCH_CHECK(max_q >= 1 && max_q < (1ll << 31) && T < (1ll << 31) && H < (1 << 16), "attention_kv8: sizes out of range");
  const bool ragged = cu.has_value() && cu->defined();
  if (ragged) {
    check_array(*cu, "cu", torch::kInt32, 1, dev);
    TORCH_CHECK(cu->size(0) == B + 1, "cu must have one entry per request and one more");
  } else {
    TORCH_CHECK(T == B && max_q == 1, "without cu every request has one query token");
  }
  const c10::cuda::CUDAGuard g(dev);
  a.q_dtype = dtype_of(q, "q", false);
  Tensor o;
  if (out.has_value() && out->defined()) {
    o = *out;
    TORCH_CHECK(o.device() == dev && o.scalar_type() == q.scalar_type() && o.is_contiguous() && o.numel() == q.numel(),
                "out must be contiguous, of q's shape and type");
  } else {
    o = torch::empty({T, H, int64_t(a.c.D)}, q.options());
  }
  Tensor lse;
  if (want_lse) lse = torch::empty({H, T}, q.options().dtype(torch::kFloat32));
  if (T == 0) return {o, lse};
  TORCH_CHECK(B >= 1, "query tokens without a request");
  a.q = q.data_ptr();
  a.q_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.table = table.data_ptr<int>();
  a.kv_len = kv_len.data_ptr<int>();
  a.cu = ragged ? cu->data_ptr<int>() : nullptr;
  a.B = int(B);
  a.T = int(T);
  a.H = int(H);
  a.width = int(table.size(1));
  a.max_q = int(max_q);
  a.scale = float(scale);
  a.o = o.data_ptr();
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  a.status = status_ptr(status, dev);
  a.num_sms = sm_count(dev.index());
  TORCH_CHECK(a.H % a.c.Hkv == 0, "heads must be a multiple of the KV heads");
  // from the caching allocator on the current stream: reused by later work of this stream only
  Tensor ws = torch::empty({int64_t(hcp::kv8::attention_workspace(a))}, q.options().dtype(torch::kUInt8));
  a.workspace = ws.data_ptr();
  HCP_CHECK_OK(hcp::kv8::attention(a, cur_stream()));
  return {o, lse};
}

Tensor sample(const Tensor& logits, const Tensor& u, optional<Tensor> t, double t_value, optional<Tensor> k, int64_t k_value,
              optional<Tensor> p, double p_value, optional<Tensor> m, double m_value, optional<Tensor> out) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "logits must be a CUDA tensor [rows, vocab] with contiguous rows");
  const auto dev = logits.device();
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 || logits.scalar_type() == torch::kBFloat16, "logits must be float32 or bfloat16");
  TORCH_CHECK(B < (1ll << 27) && V < (1ll << 31), "sample: too many rows or tokens");
  check_array(u, "u", torch::kFloat32, 1, dev);
  TORCH_CHECK(u.size(0) == B, "u must have one number per row");
  hcp::sampling::SampleArgs a{};
  auto row_f = [&](const optional<Tensor>& x, double value, const char* name) {
    hcp::sampling::RowF r{nullptr, float(value)};
    if (x.has_value() && x->defined()) {
      check_array(*x, name, torch::kFloat32, 1, dev);
      TORCH_CHECK(x->size(0) == B, name, " must have one number per row");
      r.ptr = x->data_ptr<float>();
    }
    return r;
  };
  a.temperature = row_f(t, t_value, "temperature");
  a.top_p = row_f(p, p_value, "top_p");
  a.min_p = row_f(m, m_value, "min_p");
  a.top_k = {nullptr, int(std::max<int64_t>(std::min<int64_t>(k_value, INT32_MAX), 0))};
  if (k.has_value() && k->defined()) {
    check_array(*k, "top_k", torch::kInt32, 1, dev);
    TORCH_CHECK(k->size(0) == B, "top_k must have one number per row");
    a.top_k.ptr = k->data_ptr<int>();
  }
  const c10::cuda::CUDAGuard g(dev);
  Tensor token;
  if (out.has_value() && out->defined()) {
    token = *out;
    check_array(token, "out", torch::kInt64, 1, dev);
    TORCH_CHECK(token.size(0) == B, "out must have one entry per row");
  } else {
    token = torch::empty({B}, logits.options().dtype(torch::kInt64));
  }
  a.logits = logits.data_ptr();
  a.bf16 = logits.scalar_type() == torch::kBFloat16;
  a.row_stride = logits.stride(0);
  a.B = int(B);
  a.V = int(V);
  a.u = u.data_ptr<float>();
  a.token = reinterpret_cast<long long*>(token.data_ptr<int64_t>());
  a.num_sms = sm_count(dev.index());
  HCP_CHECK_OK(hcp::sampling::sample(a, cur_stream()));
  return token;
}

}  // namespace

void bind_paged(py::module& m) {
  m.def("plan_step", &plan_step);
  m.def("rope_append_kv8", &rope_append_kv8);
  m.def("gather_kv8", &gather_kv8);
  m.def("attention_kv8", &attention_kv8);
  m.def("sample", &sample);
}
