// Python bindings of the 8-bit paged KV cache kernels.  Shapes, dtypes, devices, strides
// and alignment are checked here; page ids and lengths, which live on the device, are
// checked in the kernels and reported through the per-device error word.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include "paged8.h"

int* cfb_err_ptr(int device);
int cfb_num_sms(int device);

namespace {

using torch::Tensor;

Tensor empty(at::IntArrayRef sizes, torch::ScalarType dtype, const Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

void same_device(const Tensor& t, const Tensor& codes, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == codes.get_device(), name,
              " must be on the cache's CUDA device");
}

// codes [(layers,) P, Hkv, 2, 16, D], scales [(layers,) P, Hkv, 2]
cfb::P8Cache cache_of(const Tensor& codes, const Tensor& scales, bool layered) {
  const int64_t lead = layered ? 1 : 0;
  TORCH_CHECK(codes.is_cuda(), "codes must be a CUDA tensor");
  TORCH_CHECK(codes.dim() == 5 + lead, "codes must be ", layered ? "[layers, " : "[",
              "pages, kv_heads, 2, 16, head_dim]");
  TORCH_CHECK(codes.scalar_type() == torch::kChar ||
                  codes.scalar_type() == torch::kFloat8_e4m3fn,
              "codes must be int8 or float8_e4m3fn");
  TORCH_CHECK(codes.is_contiguous() && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
              "codes must be contiguous and 16-byte aligned");
  const int64_t D = codes.size(lead + 4);
  TORCH_CHECK(codes.size(lead + 2) == 2 && codes.size(lead + 3) == cfb::kP8Page,
              "codes must hold K and V of ", cfb::kP8Page, "-token pages");
  TORCH_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128, got ", D);
  TORCH_CHECK(codes.size(lead) >= 1 && codes.size(lead) <= 0x7fffffff &&
                  codes.size(lead + 1) >= 1 && codes.size(lead + 1) <= 65535,
              "bad page or head count");
  same_device(scales, codes, "scales");
  TORCH_CHECK(scales.scalar_type() == torch::kFloat32 && scales.is_contiguous() &&
                  scales.dim() == 3 + lead && reinterpret_cast<uintptr_t>(scales.data_ptr()) % 8 == 0,
              "scales must be contiguous fp32 [.., pages, kv_heads, 2]");
  for (int64_t i = 0; i < 3 + lead; ++i)
    TORCH_CHECK(scales.size(i) == codes.size(i), "scales do not match codes");
  cfb::P8Cache c;
  c.codes = static_cast<uint8_t*>(codes.data_ptr());
  c.scales = scales.data_ptr<float>();
  c.num_pages = codes.size(lead);
  c.Hkv = static_cast<int>(codes.size(lead + 1));
  c.D = static_cast<int>(D);
  c.fmt = codes.scalar_type() == torch::kChar ? cfb::kP8Int8 : cfb::kP8E4m3;
  return c;
}

const int32_t* ints(const Tensor& t, const Tensor& codes, int64_t dim, const char* name) {
  same_device(t, codes, name);
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.dim() == dim, name,
              " must be a contiguous ", dim, "-D int32 tensor");
  return t.data_ptr<int32_t>();
}

cfb::P8Seqs seqs_of(const Tensor& codes, const Tensor& table, const Tensor& kv_lens,
                    const c10::optional<Tensor>& cu_q) {
  cfb::P8Seqs s;
  s.table = ints(table, codes, 2, "page_table");
  s.kv_lens = ints(kv_lens, codes, 1, "kv_lens");
  TORCH_CHECK(table.size(0) == kv_lens.size(0), "page_table and kv_lens disagree");
  TORCH_CHECK(table.size(0) <= 65535, "at most 65535 sequences");
  TORCH_CHECK(table.size(1) >= 1 && table.size(1) <= (1 << 26), "bad page_table width");
  s.num_seqs = static_cast<int>(table.size(0));
  s.max_pages = static_cast<int>(table.size(1));
  if (cu_q.has_value()) {
    s.cu_q = ints(*cu_q, codes, 1, "cu_q");
    TORCH_CHECK(cu_q->size(0) == table.size(0) + 1, "cu_q must have one entry more than kv_lens");
  }
  return s;
}

int type_of(torch::ScalarType t, const char* name) {
  TORCH_CHECK(t == torch::kBFloat16 || t == torch::kHalf, name, " must be bfloat16 or float16");
  return t == torch::kBFloat16 ? cfb::kP8Bf16 : cfb::kP8Half;
}

// [N, H, D] whose rows of H * D elements are dense, 16-byte aligned and any distance apart that
// keeps them disjoint (a slice of a fused projection is one; TMA takes no expanded rows); other
// layouts are copied.
Tensor rows_of(const Tensor& t, const Tensor& codes, int64_t D, const char* name) {
  same_device(t, codes, name);
  TORCH_CHECK(t.dim() == 3 && t.size(2) == D, name, " must be [tokens, heads, ", D, "]");
  TORCH_CHECK(t.size(0) <= 0x7fffffff, name, ": too many tokens");
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()),
              "the 8-bit KV cache operators have no gradient; call them under torch.no_grad()");
  const bool dense = t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == D) &&
                     (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) * D)) &&
                     reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return dense ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t row_stride(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, " ",
              rc > 0 ? cudaGetErrorString(static_cast<cudaError_t>(rc)) : "(too large)");
}

float* mass_of(const Tensor& m, const Tensor& codes, int64_t lead, const char* name) {
  same_device(m, codes, name);
  TORCH_CHECK(m.scalar_type() == torch::kFloat32 && m.is_contiguous() && m.dim() == 3 + lead &&
                  m.size(lead + 2) == cfb::kP8Page,
              name, " must be contiguous fp32 [.., pages, kv_heads, 16]");
  for (int64_t i = 0; i < 2 + lead; ++i)
    TORCH_CHECK(m.size(i) == codes.size(i), name, " does not match codes");
  return m.data_ptr<float>();
}

void paged8_append(const Tensor& k_in, const Tensor& v_in, const Tensor& codes, const Tensor& scales,
                   const Tensor& table, const Tensor& cu_q, const Tensor& kv_lens,
                   int64_t max_q_len, const c10::optional<Tensor>& mass) {
  const cfb::P8Cache c = cache_of(codes, scales, false);
  const cfb::P8Seqs s = seqs_of(codes, table, kv_lens, cu_q);
  const Tensor k = rows_of(k_in, codes, c.D, "k"), v = rows_of(v_in, codes, c.D, "v");
  TORCH_CHECK(k.size(1) == c.Hkv && k.sizes() == v.sizes(), "k and v must be [tokens, ", c.Hkv,
              ", ", c.D, "]");
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k and v must have one dtype");
  TORCH_CHECK(max_q_len >= 1 && max_q_len <= (1 << 30), "max_q_len must be positive");
  const int type = type_of(k.scalar_type(), "k and v");
  float* m = mass.has_value() ? mass_of(*mass, codes, 0, "mass") : nullptr;
  const c10::cuda::CUDAGuard g(codes.device());
  check_rc(cfb::p8_append(c, s, k.data_ptr(), row_stride(k), v.data_ptr(), row_stride(v),
                          k.size(0),
                          static_cast<int>(max_q_len), type, m, cfb_err_ptr(codes.get_device()),
                          at::cuda::getCurrentCUDAStream()),
           "paged8_append");
}

std::tuple<Tensor, Tensor> paged8_read(const Tensor& codes, const Tensor& scales,
                                       const Tensor& table, const Tensor& kv_lens,
                                       torch::ScalarType dtype) {
  const bool layered = codes.dim() == 6;
  const cfb::P8Cache c = cache_of(codes, scales, layered);
  const cfb::P8Seqs s = seqs_of(codes, table, kv_lens, c10::nullopt);
  const int64_t layers = layered ? codes.size(0) : 1;
  TORCH_CHECK(layers <= 65535, "too many layers");
  const int type = type_of(dtype, "dtype");
  const c10::cuda::CUDAGuard g(codes.device());
  const int64_t L = static_cast<int64_t>(s.max_pages) * cfb::kP8Page;
  const auto make = [&] {
    return layered ? empty({layers, s.num_seqs, c.Hkv, L, c.D}, dtype, codes)
                   : empty({s.num_seqs, c.Hkv, L, c.D}, dtype, codes);
  };
  Tensor k = make(), v = make();
  check_rc(cfb::p8_read(c, s, static_cast<int>(layers), k.data_ptr(), v.data_ptr(), type,
                        cfb_err_ptr(codes.get_device()), at::cuda::getCurrentCUDAStream()),
           "paged8_read");
  return {k, v};
}

Tensor paged8_attention(const Tensor& q_in, const Tensor& codes, const Tensor& scales,
                        const Tensor& table, const Tensor& cu_q, const Tensor& kv_lens,
                        const c10::optional<Tensor>& out_in, double scale, int64_t max_q_len,
                        const c10::optional<Tensor>& mass_in,
                        const c10::optional<Tensor>& mass_out, int64_t workspace_bytes) {
  const cfb::P8Cache c = cache_of(codes, scales, false);
  const cfb::P8Seqs s = seqs_of(codes, table, kv_lens, cu_q);
  cfb::P8Attn a;
  const Tensor q = rows_of(q_in, codes, c.D, "q");
  a.q_stride = row_stride(q);
  a.type = type_of(q.scalar_type(), "q");
  const int64_t Hq = q.size(1), N = q.size(0);
  TORCH_CHECK(Hq >= 1 && Hq % c.Hkv == 0, "query heads (", Hq, ") must be a multiple of KV heads (",
              c.Hkv, ")");
  const c10::cuda::CUDAGuard g(codes.device());
  const Tensor out = out_in.has_value() ? *out_in : empty({N, Hq, c.D}, q.scalar_type(), codes);
  same_device(out, codes, "out");
  TORCH_CHECK(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() &&
                  out.is_contiguous() && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "out must be contiguous, like q");
  TORCH_CHECK(max_q_len >= 1 && max_q_len * (Hq / c.Hkv) < (1ll << 30), "bad max_q_len");
  TORCH_CHECK(mass_in.has_value() == mass_out.has_value(), "mass needs both input and output");
  TORCH_CHECK(scale > 0 && scale <= 3e38, "scale must be positive and finite");
  if (mass_out.has_value()) {
    a.mass_in = mass_of(*mass_in, codes, 0, "mass");
    a.mass_out = mass_of(*mass_out, codes, 0, "mass_out");
  }
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.N = N;
  a.Hq = static_cast<int>(Hq);
  a.max_q_len = static_cast<int>(max_q_len);
  a.scale = static_cast<float>(scale);
  if (s.num_seqs == 0 || (N == 0 && a.mass_out == a.mass_in)) return out;
  if (N == 0) {  // no rows, but the cached tokens' weights go on to mass_out
    a.Hq = c.Hkv;
    a.max_q_len = 1;
  }
  const int sms = cfb_num_sms(codes.get_device()), group = a.Hq / c.Hkv;
  int* err = cfb_err_ptr(codes.get_device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  const bool mass = a.mass_out != nullptr;
  TORCH_CHECK(group <= 128, "at most 128 query heads for each KV head");
  TORCH_CHECK(s.num_seqs * static_cast<int64_t>(c.Hkv) <= 65535 &&
                  c.num_pages * c.Hkv <= 0x7fffffff,
              "too many sequences or pages");
  if (!cfb::p8_is_chunk(a.max_q_len, group)) {
    // sequences at a time, within the workspace limit: kept scores are as long as the table is wide
    cfb::P8Seqs part = s;
    cfb::P8AttnPlan plan = cfb::p8_attn_plan(c, part, group, a.max_q_len, mass, sms);
    while (part.num_seqs > 1 && plan.floats() > workspace_bytes / 4) {
      part.num_seqs = (part.num_seqs + 1) / 2;
      plan = cfb::p8_attn_plan(c, part, group, a.max_q_len, mass, sms);
    }
    const int seqs_each = part.num_seqs;
    Tensor ws;
    if (plan.floats() > 0) ws = empty({plan.floats()}, torch::kFloat32, codes);
    for (int64_t i = 0; i < s.num_seqs; i += seqs_each) {
      part.table = s.table + i * s.max_pages;
      part.cu_q = s.cu_q + i;
      part.kv_lens = s.kv_lens + i;
      part.num_seqs = static_cast<int>(std::min<int64_t>(seqs_each, s.num_seqs - i));
      check_rc(cfb::p8_attention(c, part, a, plan,
                                 plan.floats() > 0 ? ws.data_ptr<float>() : nullptr, err, stream),
               "paged8_attention");
    }
    return out;
  }
  const int64_t blocks = cfb::p8_chunk_blocks(s);
  const int64_t each = static_cast<int64_t>(c.Hkv) * blocks * cfb::kP8Page * c.D;
  // sequences expanded at a time, within the workspace limit
  const int64_t seqs_each =
      std::max<int64_t>(1, std::min<int64_t>(s.num_seqs, workspace_bytes / (4 * each)));
  cfb::p8_chunk_plan(s, c.Hkv, group, a.max_q_len, sms, &a.chunk_nq, &a.splits);
  if (seqs_each < s.num_seqs) a.splits = 1;
  a.num_sms = sms;
  // one workspace: expanded K | V | their block scales | split outputs | log-sum-exps | totals
  const int64_t n_kv = seqs_each * each / 2;  // floats
  const int64_t n_par = seqs_each * c.Hkv * blocks * 4;
  const int64_t n_o = a.splits > 1 ? N * Hq * a.splits * c.D : 0;
  const int64_t n_lse = a.splits > 1 || mass ? N * Hq * a.splits : 0;
  const int64_t n_total = a.splits > 1 && mass ? N * Hq : 0;
  const Tensor ws = empty({2 * n_kv + n_par + n_o + n_lse + n_total}, torch::kFloat32, codes);
  float* at = ws.data_ptr<float>();
  a.ws_k = at;
  a.ws_v = at + n_kv;
  a.ws_par = at + 2 * n_kv;
  at += 2 * n_kv + n_par;
  a.ws_o = n_o ? at : nullptr;
  a.ws_lse = n_lse ? at + n_o : nullptr;
  a.ws_total = n_total ? at + n_o + n_lse : nullptr;
  for (int64_t i = 0; i < s.num_seqs; i += seqs_each) {
    cfb::P8Seqs part = s;
    part.table += i * s.max_pages;
    part.cu_q += i;
    part.kv_lens += i;
    part.num_seqs = static_cast<int>(std::min<int64_t>(seqs_each, s.num_seqs - i));
    check_rc(cfb::p8_chunk_attention(c, part, a, err, stream), "paged8_attention");
  }
  return out;
}

Tensor paged8_evict(const Tensor& codes, const Tensor& scales, const Tensor& mass,
                    const Tensor& table, const Tensor& kv_lens, const Tensor& dst_table,
                    int64_t budget, int64_t recent) {
  const bool layered = codes.dim() == 6;
  const cfb::P8Cache c = cache_of(codes, scales, layered);
  const cfb::P8Seqs s = seqs_of(codes, table, kv_lens, c10::nullopt);
  const int64_t layers = layered ? codes.size(0) : 1;
  float* m = mass_of(mass, codes, layered ? 1 : 0, "mass");
  const int32_t* dst = ints(dst_table, codes, 2, "dst_table");
  TORCH_CHECK(budget >= 1 && budget <= (1 << 30) && recent >= 0 && recent <= budget,
              "need 0 <= recent <= budget and budget >= 1");
  TORCH_CHECK(dst_table.size(0) == s.num_seqs && dst_table.size(1) >= 1 &&
                  dst_table.size(1) <= (1 << 26),
              "dst_table must have one row for each sequence");
  TORCH_CHECK(layers <= 65535, "too many layers");
  const c10::cuda::CUDAGuard g(codes.device());
  const Tensor keep = layered
                          ? empty({layers, s.num_seqs, c.Hkv, budget}, torch::kInt32, codes)
                          : empty({s.num_seqs, c.Hkv, budget}, torch::kInt32, codes);
  check_rc(cfb::p8_evict(c, s, m, static_cast<int>(layers), dst,
                         static_cast<int>(dst_table.size(1)), static_cast<int>(budget),
                         static_cast<int>(recent), keep.data_ptr<int32_t>(),
                         cfb_err_ptr(codes.get_device()), at::cuda::getCurrentCUDAStream()),
           "paged8_evict");
  return keep;
}

}  // namespace

void register_paged8(pybind11::module& m) {
  m.def("paged8_append", &paged8_append);
  m.def("paged8_read", &paged8_read);
  m.def("paged8_attention", &paged8_attention);
  m.def("paged8_evict", &paged8_evict);
}
