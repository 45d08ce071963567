// sy_torch.cpp -- the thin PyTorch C++ extension over the C ABI.
//
// The Python autograd functions of switchyard.triton_op (forward and backward
// of _BlockAttnResTriton, src/switchyard/triton_op.py:504-589 in the
// reference) call these instead of several Python-level steps: one call does
// the output/statistics/partial-row allocations (torch's caching allocator, on
// the tensor's device and its current stream), the launches through
// include/switchyard_b200.h, and the status check. Arguments arrive already
// validated by the Python layer (which keeps the reference's exception types
// and messages); only the invariants the kernels rely on are checked here.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

#include "switchyard_b200.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16:
      return SY_BF16;
    case at::kHalf:
      return SY_F16;
    case at::kFloat:
      return SY_F32;
    default:
      TORCH_CHECK(false, "switchyard kernels take bfloat16, float16 or float32 tensors, got ", t);
  }
  return -1;
}

void check(int status, const char* what) {
  TORCH_CHECK(status == SY_OK, "switchyard: ", what, " failed (status ", status,
              "): ", sy_status_string(status));
}

sy_stream_t stream_of(const at::Tensor& t) {
  return static_cast<sy_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void need_cuda_contiguous(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.is_contiguous(), "switchyard: ", name,
              " must be a contiguous CUDA tensor");
}

// out [B, T, D] in v's dtype and the fp32 statistics [B*T, SW], plus the kernel
// family the planner picked (sy_plan_kind; -1 when nothing was launched).
std::tuple<at::Tensor, at::Tensor, int64_t> forward(const at::Tensor& v, const at::Tensor& w,
                                                    double eps) {
  need_cuda_contiguous(v, "v");
  need_cuda_contiguous(w, "w");
  TORCH_CHECK(v.dim() == 4 && w.dim() == 1 && w.size(0) == v.size(3), "switchyard: bad shapes");
  const c10::cuda::CUDAGuard guard(v.device());
  const int64_t n = v.size(0), b = v.size(1), t = v.size(2), d = v.size(3), bt = b * t;
  at::Tensor out = at::empty({b, t, d}, v.options());
  at::Tensor stats = at::empty({bt, sy_stats_stride(n)}, v.options().dtype(at::kFloat));
  int64_t kind = -1;
  if (bt > 0 && d > 0) {
    const int vd = dtype_code(v.scalar_type());
    check(sy_fwd(v.data_ptr(), w.data_ptr(), out.data_ptr(), stats.data_ptr<float>(), n, bt, d,
                 vd, dtype_code(w.scalar_type()), static_cast<float>(eps), stream_of(v)),
          "sy_fwd");
    kind = sy_plan_kind(0, n, bt, d, 1, vd);
  }
  return {out, stats, kind};
}

// dv [N, B, T, D] and the fp32 dw partial rows [P, D] (undefined when D == 0).
std::tuple<at::Tensor, at::Tensor> backward_partials(const at::Tensor& v, const at::Tensor& w,
                                                     const at::Tensor& stats,
                                                     const at::Tensor& grad_out, double eps) {
  need_cuda_contiguous(v, "v");
  need_cuda_contiguous(w, "w");
  need_cuda_contiguous(stats, "stats");
  const c10::cuda::CUDAGuard guard(v.device());
  const at::Tensor g = grad_out.to(v.scalar_type()).contiguous();
  const int64_t n = v.size(0), bt = v.size(1) * v.size(2), d = v.size(3);
  TORCH_CHECK(g.numel() == bt * d, "switchyard: gradient of the wrong size");
  at::Tensor dv = at::empty_like(v);
  if (d == 0) return {dv, at::Tensor()};
  const int vd = dtype_code(v.scalar_type());
  const int64_t p = sy_bwd_partials(n, bt, d, vd);
  TORCH_CHECK(p >= 1, "switchyard: sy_bwd_partials failed (status ", -p, "): ",
              sy_status_string(static_cast<int>(-p)));
  at::Tensor part = at::empty({p, d}, v.options().dtype(at::kFloat));
  check(sy_bwd(v.data_ptr(), w.data_ptr(), g.data_ptr(), stats.data_ptr<float>(), dv.data_ptr(),
               part.data_ptr<float>(), p, n, bt, d, vd, dtype_code(w.scalar_type()),
               static_cast<float>(eps), stream_of(v)),
        "sy_bwd");
  return {dv, part};
}

// dv and dw = the fixed-order sum of the partial rows, in `dw_dtype`.
std::tuple<at::Tensor, at::Tensor> backward(const at::Tensor& v, const at::Tensor& w,
                                            const at::Tensor& stats, const at::Tensor& grad_out,
                                            double eps, at::ScalarType dw_dtype) {
  auto [dv, part] = backward_partials(v, w, stats, grad_out, eps);
  const c10::cuda::CUDAGuard guard(v.device());
  at::Tensor dw = at::empty({w.size(0)}, w.options().dtype(dw_dtype));
  if (part.defined())
    check(sy_dw_reduce(part.data_ptr<float>(), part.size(0), part.size(1), dw.data_ptr(),
                       dtype_code(dw_dtype), stream_of(v)),
          "sy_dw_reduce");
  return {dv, dw};
}

// With the module's gain, q = w * gain: dv, and dw = dq * gain, dgain = dq * w
// in one reduction launch (either may be skipped: undefined tensor returned).
std::tuple<at::Tensor, at::Tensor, at::Tensor> backward_gain(
    const at::Tensor& v, const at::Tensor& q, const at::Tensor& stats, const at::Tensor& grad_out,
    const at::Tensor& w, const at::Tensor& gain, double eps, bool need_dw, bool need_dg) {
  need_cuda_contiguous(w, "w");
  need_cuda_contiguous(gain, "gain");
  auto [dv, part] = backward_partials(v, q, stats, grad_out, eps);
  const c10::cuda::CUDAGuard guard(v.device());
  at::Tensor dw = need_dw ? at::empty_like(w) : at::Tensor();
  at::Tensor dg = need_dg ? at::empty_like(gain) : at::Tensor();
  if (!part.defined()) {
    if (need_dw) dw.zero_();
    if (need_dg) dg.zero_();
  } else if (need_dw || need_dg) {
    check(sy_dw_reduce_gain(part.data_ptr<float>(), part.size(0), part.size(1), w.data_ptr(),
                            gain.data_ptr(), need_dw ? dw.data_ptr() : nullptr,
                            need_dg ? dg.data_ptr() : nullptr, dtype_code(w.scalar_type()),
                            stream_of(v)),
          "sy_dw_reduce_gain");
  }
  return {dv, dw, dg};
}

// ---------------------------------------------------------------------------
// serving: the arguments are checked here, so a call is one step from Python
// ---------------------------------------------------------------------------

using OptTensor = std::optional<at::Tensor>;

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

void no_grad(std::initializer_list<const at::Tensor*> ts, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->requires_grad(), what, " has no backward; run it under torch.no_grad()");
}

void same_device(const at::Tensor& t, const at::Tensor& as, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.device() == as.device(), "every input must be on the same CUDA device, ", name,
                    " is on ", t.device(), " and not on ", as.device());
}

void need_dtype(const at::Tensor& t, at::ScalarType type, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}

int serving_dtype(const at::Tensor& t) {
  const at::ScalarType s = t.scalar_type();
  TORCH_CHECK_VALUE(s == at::kBFloat16 || s == at::kHalf || s == at::kFloat,
                    "switchyard kernels take bfloat16, float16 or float32 tensors, got ", s);
  return dtype_code(s);
}

// a vector the kernels read without strides
at::Tensor index_vector(const at::Tensor& t, int64_t n, at::ScalarType type, const at::Tensor& as,
                        const char* name) {
  same_device(t, as, name);
  need_dtype(t, type, name);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " must be [", n, "], got ", shape_of(t));
  return t.contiguous();
}

// The two caches [pages, kv_heads, page_size, head_dim]; they are written or
// read in place, so they are never copied.
void check_caches(const at::Tensor& kc, const at::Tensor& vc) {
  TORCH_CHECK_VALUE(kc.dim() == 4 && vc.dim() == 4 && kc.sizes() == vc.sizes(),
                    "k_cache and v_cache must be [pages, kv_heads, page_size, head_dim], got ",
                    shape_of(kc), " and ", shape_of(vc));
  TORCH_CHECK_VALUE(kc.is_cuda(), "k_cache must be a CUDA tensor");
  same_device(vc, kc, "v_cache");
  TORCH_CHECK_VALUE(kc.scalar_type() == vc.scalar_type(),
                    "k_cache and v_cache must have the same dtype");
  TORCH_CHECK_VALUE(kc.size(1) > 0 && kc.size(2) > 0 && kc.size(3) > 0,
                    "kv_heads, page_size and head_dim must be positive");
  TORCH_CHECK_VALUE((kc.size(3) == 1 || (kc.stride(3) == 1 && vc.stride(3) == 1)),
                    "the caches' last dimension must be contiguous");
}

at::Tensor last_contiguous(const at::Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// Rows of 16-bit elements that all start at multiples of 16 bytes (an axis of one
// element may carry any stride).
bool rows_aligned(const at::Tensor& t) {
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % 8) return false;
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// Rotated q (undefined without q); the caches are written.
OptTensor append_kv(const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& kc,
                    const at::Tensor& vc, const at::Tensor& slots_in, const OptTensor& q_in,
                    const OptTensor& pos_in, const OptTensor& cos_in, const OptTensor& sin_in) {
  check_caches(kc, vc);
  no_grad({&k_in, &v_in, &kc, &vc}, "append_kv");
  if (q_in) no_grad({&*q_in}, "append_kv");
  const int64_t hk = kc.size(1), d = kc.size(3);
  sy_append_kv_args a = {};
  a.dtype = serving_dtype(kc);
  auto heads = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == d, name, " must be [tokens, heads, ", d,
                      "], got ", shape_of(t));
    same_device(t, kc, name);
    TORCH_CHECK_VALUE(t.scalar_type() == kc.scalar_type(), name,
                      " must have the same dtype as the caches");
    return last_contiguous(t);
  };
  const at::Tensor k = heads(k_in, "k"), v = heads(v_in, "v");
  const int64_t t = k.size(0);
  TORCH_CHECK_VALUE(k.size(1) == hk && v.size(1) == hk && v.size(0) == t,
                    "k and v must be [tokens, ", hk, ", ", d, "], got ", shape_of(k), " and ",
                    shape_of(v));
  const at::Tensor slots = index_vector(slots_in, t, at::kLong, kc, "slots");
  const c10::cuda::CUDAGuard guard(kc.device());
  at::Tensor q, q_out, pos, cos, sin;
  if (q_in) {
    q = heads(*q_in, "q");
    TORCH_CHECK_VALUE(q.size(0) == t, "q must be [", t, ", heads, ", d, "], got ", shape_of(q));
    q_out = at::empty({t, q.size(1), d}, q.options());
    a.q = q.data_ptr(), a.q_out = q_out.data_ptr();
    a.q_heads = q.size(1), a.q_tok = q.stride(0), a.q_head = q.stride(1);
  }
  TORCH_CHECK_VALUE(pos_in.has_value() == cos_in.has_value() &&
                        pos_in.has_value() == sin_in.has_value(),
                    "positions, cos and sin come together");
  if (pos_in) {
    pos = index_vector(*pos_in, t, at::kInt, kc, "positions");
    TORCH_CHECK_VALUE(cos_in->dim() == 2 && cos_in->sizes() == sin_in->sizes(),
                      "cos and sin must be [length, rotated / 2], got ", shape_of(*cos_in), " and ",
                      shape_of(*sin_in));
    same_device(*cos_in, kc, "cos");
    same_device(*sin_in, kc, "sin");
    need_dtype(*cos_in, at::kFloat, "cos");
    need_dtype(*sin_in, at::kFloat, "sin");
    const int64_t h = cos_in->size(1);
    TORCH_CHECK_VALUE(cos_in->size(0) > 0 && h > 0 && 2 * h <= d,
                      "cos and sin must have at least one row and 1 to ", d / 2, " columns, got ",
                      shape_of(*cos_in));
    cos = cos_in->contiguous(), sin = sin_in->contiguous();
    a.positions = pos.data_ptr<int32_t>();
    a.cos = cos.data_ptr<float>(), a.sin = sin.data_ptr<float>();
    a.rot_half = h, a.rope_len = cos.size(0), a.rope_row = h;
  }
  a.k = k.data_ptr(), a.v = v.data_ptr();
  a.k_cache = kc.data_ptr(), a.v_cache = vc.data_ptr(), a.slots = slots.data_ptr<int64_t>();
  a.tokens = t, a.kv_heads = hk, a.head_dim = d;
  a.pages = kc.size(0), a.page_size = kc.size(2);
  a.k_tok = k.stride(0), a.k_head = k.stride(1), a.v_tok = v.stride(0), a.v_head = v.stride(1);
  a.kc_page = kc.stride(0), a.kc_head = kc.stride(1), a.kc_row = kc.stride(2);
  a.vc_page = vc.stride(0), a.vc_head = vc.stride(1), a.vc_row = vc.stride(2);
  check(sy_append_kv(&a, stream_of(kc)), "sy_append_kv");
  return q_in ? OptTensor(q_out) : OptTensor();
}

// out [B, Q, Hq, D] and, if asked for, lse [B, Q, Hq].
std::tuple<at::Tensor, OptTensor> attend_paged(const at::Tensor& q_in, const at::Tensor& kc,
                                               const at::Tensor& vc, const at::Tensor& table_in,
                                               const at::Tensor& lens_in,
                                               const OptTensor& prefix_in, int64_t prefix_len,
                                               std::optional<double> scale, bool want_lse) {
  check_caches(kc, vc);
  no_grad({&q_in, &kc, &vc}, "attend_paged");
  TORCH_CHECK_VALUE(q_in.dim() == 4, "q must be [batch, q_len, q_heads, head_dim], got ",
                    shape_of(q_in));
  same_device(q_in, kc, "q");
  TORCH_CHECK_VALUE(q_in.scalar_type() == kc.scalar_type(),
                    "q must have the same dtype as the caches");
  TORCH_CHECK_VALUE(kc.scalar_type() == at::kBFloat16 || kc.scalar_type() == at::kHalf,
                    "attend_paged takes bfloat16 or float16 tensors, got ", kc.scalar_type());
  const int64_t b = q_in.size(0), n = q_in.size(1), hq = q_in.size(2), d = q_in.size(3);
  const int64_t hk = kc.size(1), page = kc.size(2);
  TORCH_CHECK_VALUE(d == kc.size(3), "q and the caches must have one head_dim, got ", d, " and ",
                    kc.size(3));
  TORCH_CHECK_VALUE(hq > 0 && hq % hk == 0, "q_heads must be a positive multiple of kv_heads, got ",
                    hq, " and ", hk);
  TORCH_CHECK_VALUE(d % 8 == 0 && d <= 128, "head_dim must be a multiple of 8 up to 128, got ", d);
  TORCH_CHECK_VALUE(page % 8 == 0, "page_size must be a multiple of 8, got ", page);
  for (const at::Tensor* c : {&kc, &vc})
    TORCH_CHECK_VALUE(rows_aligned(*c), "the caches' rows must start at multiples of 16 bytes");
  TORCH_CHECK_VALUE(table_in.dim() == 2 && table_in.size(0) == b, "page_table must be [", b,
                    ", pages a sequence], got ", shape_of(table_in));
  same_device(table_in, kc, "page_table");
  need_dtype(table_in, at::kInt, "page_table");
  const at::Tensor lens = index_vector(lens_in, b, at::kInt, kc, "kv_lens");
  const at::Tensor table = last_contiguous(table_in);
  TORCH_CHECK_VALUE(!scale || (*scale <= 2.35e38 && static_cast<float>(*scale) > 0.f),
                    "scale must be positive and finite, in 32 bits and times log2(e), got ",
                    scale.value_or(0.0));
  TORCH_CHECK_VALUE(prefix_len >= 0, "prefix_len must not be negative, got ", prefix_len);
  at::Tensor prefix;
  if (prefix_len > 0) {
    TORCH_CHECK_VALUE(prefix_in.has_value(), "prefix_len ", prefix_len, " needs prefix_pages");
    same_device(*prefix_in, kc, "prefix_pages");
    need_dtype(*prefix_in, at::kInt, "prefix_pages");
    TORCH_CHECK_VALUE(prefix_in->dim() == 1 && prefix_in->size(0) >= (prefix_len + page - 1) / page,
                      "prefix_pages must hold the ", (prefix_len + page - 1) / page,
                      " pages of prefix_len ", prefix_len, ", got ", shape_of(*prefix_in));
    prefix = prefix_in->contiguous();
  }
  const c10::cuda::CUDAGuard guard(kc.device());
  at::Tensor q = q_in;
  if (q.numel() && (q.stride(3) != 1 || !rows_aligned(q)))
    q = q.clone(at::MemoryFormat::Contiguous);
  at::Tensor out = at::empty({b, n, hq, d}, q.options());
  OptTensor lse;
  if (want_lse) lse = at::empty({b, n, hq}, q.options().dtype(at::kFloat));
  sy_attend_args a = {};
  a.q = q.data_ptr(), a.k_cache = kc.data_ptr(), a.v_cache = vc.data_ptr();
  a.out = out.data_ptr(), a.lse = want_lse ? lse->data_ptr<float>() : nullptr;
  a.page_table = table.data_ptr<int32_t>(), a.kv_lens = lens.data_ptr<int32_t>();
  a.prefix_pages = prefix_len > 0 ? prefix.data_ptr<int32_t>() : nullptr;
  a.batch = b, a.q_len = n, a.q_heads = hq, a.kv_heads = hk, a.head_dim = d;
  a.pages = kc.size(0), a.page_size = page;
  a.table_width = table.size(1), a.table_row = table.stride(0), a.prefix_len = prefix_len;
  a.q_b = q.stride(0), a.q_t = q.stride(1), a.q_h = q.stride(2);
  a.kc_page = kc.stride(0), a.kc_head = kc.stride(1), a.kc_row = kc.stride(2);
  a.vc_page = vc.stride(0), a.vc_head = vc.stride(1), a.vc_row = vc.stride(2);
  a.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(d)));
  a.dtype = dtype_code(kc.scalar_type());
  const int64_t bytes = sy_attend_workspace(&a);
  TORCH_CHECK(bytes >= 0, "switchyard: sy_attend_workspace failed (status ", -bytes, "): ",
              sy_status_string(static_cast<int>(-bytes)));
  at::Tensor ws;
  if (bytes > 0) {
    ws = at::empty({bytes}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
  }
  check(sy_attend(&a, stream_of(kc)), "sy_attend");
  return {out, lse};
}

// token [rows] and, if asked for, logprob [rows].
std::tuple<at::Tensor, OptTensor> sample_tokens(const at::Tensor& logits_in, const at::Tensor& u_in,
                                                const OptTensor& temperature,
                                                const OptTensor& top_k, const OptTensor& top_p,
                                                const OptTensor& min_p, bool want_logprob) {
  TORCH_CHECK_VALUE(logits_in.dim() == 2 && logits_in.size(1) > 0,
                    "logits must be [rows, vocab], got ", shape_of(logits_in));
  TORCH_CHECK_VALUE(logits_in.is_cuda(), "logits must be a CUDA tensor");
  no_grad({&logits_in}, "sample_tokens");
  sy_sample_args a = {};
  a.dtype = serving_dtype(logits_in);
  const int64_t rows = logits_in.size(0), vocab = logits_in.size(1);
  TORCH_CHECK_VALUE(vocab <= (int64_t(1) << 22), "vocab must be at most ", int64_t(1) << 22,
                    ", got ", vocab);
  const c10::cuda::CUDAGuard guard(logits_in.device());
  at::Tensor logits = last_contiguous(logits_in);
  if (rows > 1 && logits.stride(0) < vocab) logits = logits.contiguous();
  const at::Tensor u = index_vector(u_in, rows, at::kFloat, logits, "u");
  at::Tensor keep[4];
  auto per_row = [&](const OptTensor& t, at::ScalarType type, const char* name,
                     at::Tensor& hold) -> void* {
    if (!t) return nullptr;
    hold = index_vector(*t, rows, type, logits, name);
    return hold.data_ptr();
  };
  a.temperature = static_cast<float*>(per_row(temperature, at::kFloat, "temperature", keep[0]));
  a.top_k = static_cast<int32_t*>(per_row(top_k, at::kInt, "top_k", keep[1]));
  a.top_p = static_cast<float*>(per_row(top_p, at::kFloat, "top_p", keep[2]));
  a.min_p = static_cast<float*>(per_row(min_p, at::kFloat, "min_p", keep[3]));
  at::Tensor token = at::empty({rows}, logits.options().dtype(at::kLong));
  OptTensor logprob;
  if (want_logprob) logprob = at::empty({rows}, logits.options().dtype(at::kFloat));
  a.logits = logits.data_ptr(), a.u = u.data_ptr<float>();
  a.token = token.data_ptr<int64_t>();
  a.logprob = want_logprob ? logprob->data_ptr<float>() : nullptr;
  a.rows = rows, a.vocab = vocab, a.logits_row = rows > 1 ? logits.stride(0) : vocab;
  check(sy_sample(&a, stream_of(logits)), "sy_sample");
  return {token, logprob};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "switchyard B200: PyTorch C++ extension over the C ABI of libswitchyard_b200.so";
  m.def("forward", &forward, "sy_fwd: (out, stats, plan kind)");
  m.def("backward_partials", &backward_partials, "sy_bwd: (dv, dw partial rows)");
  m.def("backward", &backward, "sy_bwd + sy_dw_reduce: (dv, dw)");
  m.def("backward_gain", &backward_gain, "sy_bwd + sy_dw_reduce_gain: (dv, dw, dgain)");
  m.def("append_kv", &append_kv, "sy_append_kv: rotated q or None");
  m.def("attend_paged", &attend_paged, "sy_attend: (out, lse or None)");
  m.def("sample_tokens", &sample_tokens, "sy_sample: (token, logprob or None)");
  m.def("version", []() { return std::string(sy_version()); });
}
